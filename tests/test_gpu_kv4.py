"""The 4-bit cache on the GPU, through madi_amd.kv4: the bytes that a store
writes (every byte of the pool compared), the values a load gives, attention
against float64 over the codes.

Tolerances.  Stores and loads are exact (a load rounds q * s once).  Attention,
per element, with E the bound on a score's error (kv4_ref.score_error), A the mean
|v| with the row's weights and n keys:
  f16 rows   P and V are rounded to f16 (2^-11 each), out once (2^-11)
  f32 rows   q, P to 22 bits (2^-22 each and the low parts' product, 2^-22), V exactly
  both       a weight is off by 2E (numerator and sum) and by exp2 (2^-21 with its
             argument's rounding at up to 2^4 .. 2^5: 32 * 2^-24); n/32 + 64
             additions of partial results; and absolutely 2^-32 sum|v|, since P
             lies on f16's finest grid: each weight is off by up to 2^-25 (with
             low parts too: their grid is the same 2^-24) where the largest P,
             so the weights' sum, is at least 2^7.  That counts where the keys
             that carry the weight have v = 0 and A is small.
and for f32 rows normwise 2e-5: the roundings of a score taken as independent
come to 1e-5 at these sizes, while a low part left out would show as 1e-4.
"""
import sys

import numpy as np
import pytest

import kv4_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def kv4():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import madi_amd.kv4 as kv4
    import madi_amd.q8 as q8
    q8.init()
    return kv4


NP = {"f16": np.float16, "f32": np.float32}


class Setup:
    """Sequences with shuffled pages in a pool of random bytes."""

    def __init__(self, kv4, rng, heads, d, page, lens, rows, spare=3, bad=()):
        self.kv4, self.heads, self.d, self.page, self.lens, self.rows = kv4, heads, d, page, lens, rows
        need = [-(-n // page) for n in lens]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages)
        self.table = rng.integers(0, 1 << 31, (len(lens), max(max(need), 1) + 1)).astype(np.int32)
        at = 0
        for i, c in enumerate(need):
            self.table[i, :c] = order[at:at + c]
            at += c
        for i, j, v in bad:
            self.table[i, j] = np.uint32(v).astype(np.int32)
        self.data = rng.integers(0, 256, (self.n_pages, heads, R.block_bytes(page, d)), dtype=np.uint8)
        off = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.m = int(off[-1])
        self.uniform = len(set(rows)) == 1
        self.dev = torch.from_numpy(self.data).cuda()
        self.cache = kv4.KV4(self.dev, page, heads, d, self.n_pages)
        self.batch = kv4.Batch(torch.from_numpy(self.table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                               rows=max(rows), row_off=None if self.uniform else torch.from_numpy(off).cuda(),
                               m=self.m)
        self.off = off

    def place(self, i, pos):
        p = int(np.uint32(self.table[i, pos // self.page]))
        return (p, pos % self.page) if p < self.n_pages else (None, 0)

    def fill(self, rng, spread=1.0):
        """Codes and scales of every token of every sequence, written into the pool."""
        self.held = []
        for i, n in enumerate(self.lens):
            k = rng.standard_normal((n, self.heads, self.d)) * spread
            k[:, :, ::17] *= 4
            v = rng.standard_normal((n, self.heads, self.d))
            kq, ks = R.quantise(k.astype(np.float32))
            vq, vs = R.quantise(v.astype(np.float32))
            there = np.zeros(n, bool)
            for t in range(n):
                p, o = self.place(i, t)
                if p is None:
                    continue
                there[t] = True
                for h in range(self.heads):
                    R.put(self.data, self.page, self.d, p, h, o, kq[t, h], ks[t, h], vq[t, h], vs[t, h])
            self.held.append((kq, ks, vq, vs, there))
        self.dev.copy_(torch.from_numpy(self.data))

    def expect(self, q, nh, causal, window, scale, dtype):
        """Exact outputs and their tolerances [m][nh][d]."""
        g = nh // self.heads
        out, tol = np.zeros((self.m, nh, self.d)), np.zeros((self.m, nh, self.d))
        for i, n in enumerate(self.lens):
            kq, ks, vq, vs, there = self.held[i]
            r0, r1 = self.off[i], self.off[i + 1]
            for h in range(self.heads):
                qh = q[r0:r1, h * g:(h + 1) * g]
                o, a, v1 = R.attention(qh, R.value(kq[:, h], ks[:, h]), R.value(vq[:, h], vs[:, h]), there,
                                         list(R.rows_of(n, r1 - r0)), causal, window, scale)
                e = R.score_error(qh, ks[:, h], scale)[..., None]
                if dtype == "f16":
                    t = (2.0 ** -10 + 2 * e + 32 * 2.0 ** -23 + (n / 32 + 64) * 2.0 ** -24) * a
                    t += 2.0 ** -11 * np.abs(o) + 2.0 ** -25 + 2.0 ** -32 * v1
                else:
                    # q's own rounding is 2^-22 of |q| |k|: within E's 80 * 7 * 2^-24
                    t = (3 * 2.0 ** -22 + 2 * e + 32 * 2.0 ** -23 + (n / 32 + 64) * 2.0 ** -24) * a
                    t += 2.0 ** -24 * np.abs(o) + 2.0 ** -32 * v1
                out[r0:r1, h * g:(h + 1) * g] = o
                tol[r0:r1, h * g:(h + 1) * g] = t
        return out, tol


def attend(s, q, nh, dtype, causal=True, window=0, scale=None, reserve=True, out=None):
    tq = torch.from_numpy(q.reshape(s.m, -1)).cuda()
    to = torch.full_like(tq, 77.0) if out is None else out
    if reserve:
        s.batch.reserve(s.cache, nh)
    s.kv4.kvAttn(to, tq, s.cache, s.batch, nh, causal=causal, window=window, scale=scale)
    torch.cuda.synchronize()
    return to.cpu().numpy().reshape(s.m, nh, s.d).astype(np.float64)


def check(got, want, tol, dtype, what=""):
    assert np.all(np.isfinite(got)), what
    worst = (np.abs(got - want) / np.maximum(tol, 1e-300)).max(initial=0)
    norm = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
    say(f"  {what} worst |err| / tol {worst:.3f}, normwise {norm:.2e}")
    assert worst <= 1, worst
    if dtype == "f32":
        assert norm <= 2e-5, norm


# ------------------------------------------------------------------ store and load
def rows_for(rng, m, heads, d, dtype, kind):
    x = rng.standard_normal((m, 2, heads, d)).astype(np.float32)
    if kind == "wide":  # magnitudes over the type's range, whole blocks of 0 among them
        top = 4 if dtype == "f16" else 30
        x = x * 10.0 ** rng.integers(-8 if dtype == "f16" else -30, top, (m, 2, heads, d // 32)).repeat(32, -1)
        x[rng.random(x.shape) < 0.1] = 0
        x.reshape(m, 2, heads, -1, 32)[rng.random((m, 2, heads, d // 32)) < 0.1] = 0
    if kind == "borders":  # |x| / s a whole number and a half, or one step of x beside it
        t, s = NP[dtype], 47 / 128  # exact in f16, and so are 7 s and (2c + 1) s / 2
        c = ((2 * rng.integers(0, 7, x.shape) + 1) * (s / 2)).astype(t)
        step = rng.integers(-1, 2, x.shape)
        c = np.where(step == 0, c, np.nextafter(c, (step * 100).astype(t)))
        x = c * rng.choice([-1, 1], x.shape).astype(t)
        x[..., ::32] = 7 * s
    if kind == "special":
        for v in (np.nan, np.inf, -np.inf, -0.0, 65504.0, 2.0 ** -24):
            x[rng.random(x.shape) < 0.01] = v
    with np.errstate(over="ignore"):
        return x.astype(NP[dtype])


STORES = [
    # heads, d, page, lens, rows, dtype, kind
    (1, 64, 16, [1], [1], "f32", "normal"),
    (20, 64, 64, [57, 448, 1, 130], [1, 1, 1, 1], "f32", "normal"),
    (2, 128, 16, [5, 40, 33, 64], [3, 40, 1, 17], "f16", "normal"),
    (3, 96, 32, [70, 9], [70, 2], "f16", "wide"),
    (2, 256, 16, [18, 31], [7, 7], "f32", "wide"),
    (2, 64, 16, [33, 50], [33, 11], "f32", "borders"),
    (2, 128, 32, [33, 50], [33, 11], "f16", "borders"),
    (2, 64, 16, [30, 21], [30, 20], "f32", "special"),
    (2, 96, 16, [30, 21], [30, 20], "f16", "special"),
    (1, 64, 16, [3, 0, 6], [5, 2, 6], "f16", "normal"),  # more rows than tokens: positions below 0
    (8, 128, 256, [700, 513], [129, 1], "f16", "normal"),
]


@pytest.mark.parametrize("heads,d,page,lens,rows,dtype,kind", STORES)
def test_store_and_load(kv4, heads, d, page, lens, rows, dtype, kind):
    """Every byte of the pool after a store: the rows' own as the format says,
    the others untouched.  Then the rows read back, rows around them untouched."""
    say(f"store {heads}x{d} page {page} lens {lens} rows {rows} {dtype} {kind}")
    rng = np.random.default_rng(len(lens) * d + page + heads)
    s = Setup(kv4, rng, heads, d, page, lens, rows)
    x = rows_for(rng, s.m, heads, d, dtype, kind)
    kv = torch.from_numpy(x).cuda()  # k | v alternate, as a stacked projection leaves them
    kv4.kvStore(s.cache, s.batch, kv[:, 0], kv[:, 1].flatten(1))
    torch.cuda.synchronize()
    (kq, ks), (vq, vs) = R.quantise(x[:, 0]), R.quantise(x[:, 1])
    want = s.data.copy()
    back = np.zeros((s.m, 2, heads, d))
    for i, n in enumerate(lens):
        for r, pos in enumerate(R.rows_of(n, rows[i])):
            row = s.off[i] + r
            if pos < 0:
                continue
            p, o = s.place(i, pos)
            for h in range(heads):
                R.put(want, page, d, p, h, o, kq[row, h], ks[row, h], vq[row, h], vs[row, h])
            back[row, 0], back[row, 1] = R.value(kq[row], ks[row]), R.value(vq[row], vs[row])
    assert np.array_equal(s.dev.cpu().numpy(), want)
    out = torch.full((s.m + 2, 2, heads * d), 99.0, dtype=kv.dtype, device="cuda")
    kv4.kvLoad(s.cache, s.batch, out[1:-1, 0], out[1:-1, 1])
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(s.m + 2, 2, heads, d)
    assert np.all(got[[0, -1]] == 99)
    assert np.array_equal(got[1:-1], back.astype(NP[dtype]))


def test_rows_that_have_no_place(kv4):
    """A page number past the pool: its rows are not stored, load as zeros; so
    do rows past m; a length past the table counts as the table's reach."""
    say("rows without a place")
    rng = np.random.default_rng(5)
    s = Setup(kv4, rng, 2, 64, 16, [40, 20], [40, 20], bad=[(0, 1, 0xffffffff), (1, 0, 10 ** 6)])
    x = torch.randn(s.m, 2, 128, device="cuda")
    s.batch.lens.copy_(torch.tensor([40, 20], dtype=torch.int32))
    kv4.kvStore(s.cache, s.batch, x[:, 0], x[:, 1])
    k, v = torch.full((2, s.m, 128), 99.0, device="cuda")
    kv4.kvLoad(s.cache, s.batch, k, v)
    torch.cuda.synchronize()
    kq, ks = R.quantise(x[:, 0].cpu().numpy().reshape(s.m, 2, 64))
    want = R.value(kq, ks)
    want[16:32] = 0      # sequence 0, page 1
    want[40:56] = 0      # sequence 1, page 0
    assert np.array_equal(k.cpu().numpy().reshape(s.m, 2, 64), want.astype(np.float32))
    pool = s.dev.clone()
    # starts past m, and a length past the table
    b = kv4.Batch(s.batch.table, torch.tensor([1 << 30, -1], dtype=torch.int32).cuda(), rows=30,
                  row_off=torch.tensor([0, 5, 1 << 30], dtype=torch.int32).cuda(), m=7)
    k.fill_(99)
    kv4.kvLoad(s.cache, b, k, v)
    torch.cuda.synchronize()
    assert (k[7:] == 99).all() and not (k[:7] == 99).any()
    assert torch.equal(s.dev, pool)


# ------------------------------------------------------------------ attention
ATTN = [
    # heads, group, d, page, lens, rows, causal, window
    (1, 1, 64, 16, [1], [1], True, 0),
    (20, 1, 64, 64, [213], [1], True, 0),
    (2, 1, 64, 16, [31, 32, 33, 64, 65, 0, 127], [1] * 7, True, 0),
    (2, 4, 128, 16, [500, 3, 129, 1], [1] * 4, True, 0),
    (1, 16, 128, 32, [40, 300], [1, 1], True, 0),
    (1, 20, 64, 16, [40, 77], [1, 1], True, 0),       # more columns than a tile
    (3, 2, 96, 16, [50, 200], [1, 1], True, 0),
    (2, 5, 256, 64, [50, 200], [2, 2], True, 0),
    (2, 2, 64, 32, [90, 16, 300], [90, 7, 61], True, 0),   # prompts
    (1, 3, 128, 16, [70, 40], [70, 33], True, 24),         # windows
    (2, 1, 64, 128, [400], [1], True, 1),
    (2, 2, 64, 16, [3, 100], [6, 4], True, 0),             # rows before the first token: zeros
    (2, 2, 64, 64, [150, 37], [9, 2], False, 0),           # cross-attention
    (2, 4, 128, 64, [1000, 2100], [1, 1], True, 0),        # split over workgroups
    (1, 8, 128, 16, [1500], [37], False, 0),
    (1, 1, 96, 64, [3000], [1], True, 2000),
]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,group,d,page,lens,rows,causal,window", ATTN)
def test_attention(kv4, heads, group, d, page, lens, rows, causal, window, dtype):
    say(f"attn {heads}x{group}x{d} page {page} lens {lens} rows {rows} causal {causal} window {window} {dtype}")
    rng = np.random.default_rng(sum(lens) + d + page)
    s = Setup(kv4, rng, heads, d, page, lens, rows)
    s.fill(rng)
    nh = heads * group
    q = rng.standard_normal((s.m, nh, d)).astype(NP[dtype])
    want, tol = s.expect(q, nh, causal, window, d ** -0.5, dtype)
    got = attend(s, q, nh, dtype, causal, window)
    check(got, want, tol, dtype, "split:")
    if s.batch.work is not None:
        s.batch._c.work, s.batch._c.work_bytes = None, 0
        check(attend(s, q, nh, dtype, causal, window, reserve=False), want, tol, dtype, "one share:")


PROMPTS = [
    # heads, group, d, page, lens, rows, causal, window: enough columns to fill the device
    (16, 16, 64, 16, [230, 233], [230, 190], True, 0),
    (16, 16, 96, 32, [220, 200], [220, 200], True, 0),
    (16, 16, 128, 64, [250, 230], [230, 230], True, 0),
    (16, 16, 256, 16, [200, 217], [200, 217], True, 0),
    (16, 8, 64, 64, [400, 270, 40], [250, 270, 40], True, 70),
    (8, 32, 64, 16, [70, 129], [250, 129], True, 0),     # rows before the first token
    (16, 16, 128, 16, [193, 30], [230, 30], False, 0),
    (20, 1, 64, 64, [1100, 1024], [1100, 1000], True, 0),
]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,group,d,page,lens,rows,causal,window", PROMPTS)
def test_prompts(kv4, heads, group, d, page, lens, rows, causal, window, dtype):
    """Rows enough for the prompts' kernel; a page missing; columns past a
    tile and rows past the last sequence left alone."""
    say(f"prompt {heads}x{group}x{d} page {page} lens {lens} rows {rows} causal {causal} window {window} {dtype}")
    rng = np.random.default_rng(sum(lens) + d + page)
    s = Setup(kv4, rng, heads, d, page, lens, rows, bad=[(0, 1, 1 << 20)] if page < 64 else ())
    s.fill(rng)
    nh = heads * group
    q = rng.standard_normal((s.m, nh, d), dtype=np.float32).astype(NP[dtype])
    out = torch.full((s.m + 2, nh * d), 77.0, dtype=getattr(torch, "float16" if dtype == "f16" else "float32"),
                     device="cuda")
    want, tol = s.expect(q, nh, causal, window, d ** -0.5, dtype)
    s.kv4.kvAttn(out, torch.from_numpy(q.reshape(s.m, -1)).cuda(), s.cache, s.batch, nh, causal=causal, window=window)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert (got[s.m:] == 77).all()
    check(got[:s.m].reshape(s.m, nh, d).astype(np.float64), want, tol, dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("qs,ks,scale", [(8.0, 1.0, None), (1.0, 100.0, 0.01), (1e-4, 1.0, 30.0), (300.0, 20.0, 1e-5),
                                         (1.0, 1.0, -0.2), (1.0, 1.0, 0.0)])
def test_magnitudes(kv4, qs, ks, scale, dtype):
    """Sharp and flat softmax, rising references, small and large operands, a
    negative scale, and none at all (the mean of V)."""
    say(f"magnitudes q {qs} k {ks} scale {scale} {dtype}")
    rng = np.random.default_rng(3)
    s = Setup(kv4, rng, 2, 64, 16, [300, 41], [3, 3])
    s.fill(rng, spread=ks)
    q = (rng.standard_normal((s.m, 4, 64)) * qs).astype(NP[dtype])
    sc = 0.125 if scale is None else scale
    want, tol = s.expect(q, 4, True, 0, np.float32(sc).astype(np.float64), dtype)
    got = attend(s, q, 4, dtype, scale=scale)
    assert np.all(np.abs(got - want) <= tol), (np.abs(got - want) / tol).max()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_pages_that_are_not_there(kv4, dtype):
    """Missing pages in the middle, at the start and all of them: their keys
    are not seen, whatever the pool holds; a sequence with none gives zeros."""
    say(f"missing pages {dtype}")
    rng = np.random.default_rng(11)
    s = Setup(kv4, rng, 2, 64, 16, [100, 70, 33], [2, 2, 2],
              bad=[(0, 2, 0xffffffff), (0, 0, 1 << 20), (2, 0, 99999), (2, 1, 99999), (2, 2, 99999)])
    s.fill(rng)
    q = rng.standard_normal((s.m, 6, 64)).astype(NP[dtype])
    want, tol = s.expect(q, 6, True, 0, 0.125, dtype)
    got = attend(s, q, 6, dtype)
    check(got, want, tol, dtype)
    assert np.all(got[4:] == 0)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_what_lies_past_the_end_is_not_seen(kv4, dtype):
    """The pool past each sequence's end filled with NaN, then with infinite scales."""
    say(f"NaN past the end {dtype}")
    rng = np.random.default_rng(12)
    s = Setup(kv4, rng, 2, 128, 64, [1, 30, 63, 65], [1, 1, 1, 1])
    for fill in ((0xff, 0xff), (0x00, 0x7c)):
        s.data[..., 0::2], s.data[..., 1::2] = fill
        s.fill(np.random.default_rng(1))
        q = rng.standard_normal((s.m, 2, 128)).astype(NP[dtype])
        want, tol = s.expect(q, 2, True, 0, 128 ** -0.5, dtype)
        check(attend(s, q, 2, dtype), want, tol, dtype)


def test_outputs_in_place_and_strided(kv4):
    """out = q itself; rows inside wider ones, the rest untouched; rows past
    the last sequence left as they were."""
    say("in place, strided")
    rng = np.random.default_rng(13)
    s = Setup(kv4, rng, 2, 64, 16, [100, 70, 9], [5, 1, 3])
    s.fill(rng)
    q = rng.standard_normal((s.m, 4, 64)).astype(np.float16)
    want, tol = s.expect(q, 4, True, 0, 0.125, "f16")
    tq = torch.from_numpy(q.reshape(s.m, -1)).cuda()
    kv4.kvAttn(tq, tq, s.cache, s.batch, 4)
    torch.cuda.synchronize()
    assert np.all(np.abs(tq.cpu().numpy().reshape(q.shape) - want) <= tol)
    wide_q = torch.full((s.m, 3, 256), 9.0, dtype=torch.float16, device="cuda")
    wide_q[:, 1] = torch.from_numpy(q.reshape(s.m, -1)).cuda()
    wide_o = torch.full((s.m + 3, 2, 256), 9.0, dtype=torch.float16, device="cuda")
    kv4.kvAttn(wide_o[:, 0], wide_q[:, 1], s.cache, s.batch, 4)
    torch.cuda.synchronize()
    assert (wide_o[:, 1] == 9).all() and (wide_o[s.m:] == 9).all()
    assert np.all(np.abs(wide_o[:s.m, 0].cpu().numpy().reshape(q.shape) - want) <= tol)


def test_reruns_are_bit_identical(kv4):
    say("reruns")
    rng = np.random.default_rng(14)
    s = Setup(kv4, rng, 2, 64, 16, [3000, 70], [2, 2])
    s.fill(rng)
    q = rng.standard_normal((s.m, 4, 64)).astype(np.float32)
    a = attend(s, q, 4, "f32")
    for _ in range(3):
        assert np.array_equal(attend(s, q, 4, "f32"), a)


def test_decode_loop_in_a_graph(kv4):
    """A decoder's steps as they are used: rows stored and attended to in one
    captured graph, lengths and rows updated in place between replays; then
    two more graphs, a batch of its own each, replayed at the same time."""
    from madi_amd import q8
    say("graph")
    rng = np.random.default_rng(15)
    heads, d, nh, page = 2, 64, 4, 16
    s = Setup(kv4, rng, heads, d, page, [600, 50], [1, 1], spare=8)
    s.lens = [590, 40]
    s.fill(rng)
    dev_lens = s.batch.lens
    batches = [s.batch] + [kv4.Batch(s.batch.table, dev_lens, rows=1) for _ in range(2)]
    for b in batches:
        b.reserve(s.cache, nh)
    k, v = torch.empty(2, 2, heads * d, device="cuda")
    q = torch.empty(2, nh * d, device="cuda")
    outs = [torch.empty_like(q) for _ in batches]
    graphs = []
    torch.cuda.synchronize()
    for i, batch in enumerate(batches):
        st = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            q8.init(st)
            if i == 0:
                kv4.kvStore(s.cache, batch, k, v)
            kv4.kvAttn(outs[i], q, s.cache, batch, nh)
        graphs.append((g, st))
    q8.init()
    for stepno in range(4):
        lens = [591 + stepno, 41 + stepno]
        kn, vn = rng.standard_normal((2, 2, heads, d)).astype(np.float32)
        qn = rng.standard_normal((2, nh, d)).astype(np.float32)
        k.copy_(torch.from_numpy(kn.reshape(2, -1)))
        v.copy_(torch.from_numpy(vn.reshape(2, -1)))
        q.copy_(torch.from_numpy(qn.reshape(2, -1)))
        dev_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        graphs[0][0].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            new = (*R.quantise(kn[i]), *R.quantise(vn[i]), np.array(True))
            s.held[i] = tuple(np.concatenate([a, b[None]]) for a, b in zip(s.held[i], new))
        s.lens = lens
        want, tol = s.expect(qn, nh, True, 0, 0.125, "f32")
        eager = torch.empty_like(q)
        kv4.kvAttn(eager, q, s.cache, s.batch, nh)
        torch.cuda.synchronize()
        for g, st in graphs[1:]:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        check(outs[0].cpu().numpy().reshape(2, nh, d).astype(np.float64), want, tol, "f32", f"step {stepno}")
        assert all(torch.equal(o, eager) for o in outs)


def test_a_pool_past_4_gib(kv4):
    """Pages whose bytes start beyond 32 bits."""
    say("large pool")
    rng = np.random.default_rng(16)
    heads, d, page = 8, 128, 256
    n_pages = (5 << 30) // (heads * R.block_bytes(page, d))
    cache = kv4.alloc(n_pages, page, heads, d)
    table = torch.tensor([[n_pages - 1, 0, n_pages - 2]], dtype=torch.int32).cuda()
    n = 600
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    x = rng.standard_normal((n, 2, heads, d)).astype(np.float16)
    kv = torch.from_numpy(x).cuda()
    b = kv4.Batch(table, lens, rows=n)
    kv4.kvStore(cache, b, kv[:, 0], kv[:, 1])
    k, v = torch.empty(2, n, heads * d, dtype=torch.float16, device="cuda")
    kv4.kvLoad(cache, b, k, v)
    torch.cuda.synchronize()
    held = [R.quantise(x[:, j]) for j in (0, 1)]
    assert np.array_equal(k.cpu().numpy().reshape(n, heads, d), R.value(*held[0]).astype(np.float16))
    assert np.array_equal(v.cpu().numpy().reshape(n, heads, d), R.value(*held[1]).astype(np.float16))
    s = Setup.__new__(Setup)
    s.kv4, s.heads, s.d, s.lens, s.m, s.off = kv4, heads, d, [n], 1, [0, 1]
    s.cache, s.batch = cache, kv4.Batch(table, lens, rows=1)
    s.held = [(*held[0], *held[1], np.ones(n, bool))]
    q = rng.standard_normal((1, heads, d)).astype(np.float16)
    want, tol = s.expect(q, heads, True, 0, 128 ** -0.5, "f16")
    check(attend(s, q, heads, "f16"), want, tol, "f16")
