"""The 4-bit cache as a server uses it: long and many sequences whose steps are
shared by the workgroups, lists of pages that are renewed on the way, small
workspaces, pages shared by sequences, rows cut off by the batch, calls on two streams and
graphs replayed at the same time.  The cache is filled by kvStore itself;
the oracle and the tolerances are those of test_gpu_kv4.py."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import NP, Setup, attend, check, kv4, say  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


class Stored(Setup):
    """A Setup whose tokens are stored by the library."""

    def fill(self, rng):
        self.held = []
        off = np.concatenate([[0], np.cumsum(self.lens)]).astype(np.int32)
        x = rng.standard_normal((int(off[-1]), 2, self.heads, self.d), dtype=np.float32).astype(np.float16)
        x[:, 0, :, ::17] *= 4
        kv = torch.from_numpy(x).cuda()
        b = self.kv4.Batch(self.batch.table, self.batch.lens, rows=max(self.lens),
                           row_off=torch.from_numpy(off).cuda(), m=int(off[-1]))
        self.kv4.kvStore(self.cache, b, kv[:, 0], kv[:, 1])
        torch.cuda.synchronize()
        for i, n in enumerate(self.lens):
            own = x[off[i]:off[i + 1]]
            there = np.array([self.place(i, t)[0] is not None for t in range(n)], bool)
            self.held.append((*R.quantise(own[:, 0]), *R.quantise(own[:, 1]), there))


def queries(rng, s, nh, dtype):
    return rng.standard_normal((s.m, nh, s.d), dtype=np.float32).astype(NP[dtype])


LONG = [
    # heads, group, d, page, lens, rows, causal, window
    (1, 2, 64, 16, [20011], [1], True, 0),          # 40 steps per wave of one workgroup: its list is renewed
    (2, 1, 128, 64, [9000, 17], [1, 1], True, 0),   # the same with 8 waves (f32)
    (1, 1, 96, 16, [17001], [2], False, 0),
    (1, 4, 256, 128, [9100], [1], True, 9000),      # a window: the steps begin past 0
]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,group,d,page,lens,rows,causal,window", LONG)
def test_long_caches_by_workspace(kv4, heads, group, d, page, lens, rows, causal, window, dtype):
    """The same rows with the full workspace, with one for five workgroups and
    with none; a page in the middle is missing."""
    say(f"long {heads}x{group}x{d} page {page} lens {lens} {dtype}")
    rng = np.random.default_rng(lens[0])
    s = Stored(kv4, rng, heads, d, page, lens, rows, bad=[(0, 3000 // page, 1 << 30)])
    s.fill(rng)
    nh = heads * group
    q = queries(rng, s, nh, dtype)
    want, tol = s.expect(q, nh, causal, window, d ** -0.5, dtype)
    check(attend(s, q, nh, dtype, causal, window), want, tol, dtype, "all:")
    part = 2 * 16 * (d + 2) * 4
    full = s.batch._c.work_bytes
    starts = full % part
    assert full > 6 * part
    for groups in (5, 1, 0):  # (one place is no sharing)
        s.batch._c.work_bytes = starts + groups * part + part // 2
        check(attend(s, q, nh, dtype, causal, window, reserve=False), want, tol, dtype, f"{groups}:")
    s.batch._c.work, s.batch._c.work_bytes = None, 0
    check(attend(s, q, nh, dtype, causal, window, reserve=False), want, tol, dtype, "none:")


def test_many_ragged_sequences(kv4):
    """More items than a scan of 64 takes, of two column tiles each, lengths
    from none to thousands, sequences without rows among them; the workspace starts as NaN."""
    say("many")
    rng = np.random.default_rng(21)
    heads, d, nh = 2, 64, 8
    lens = [int(n) for n in rng.integers(0, 300, 75)]
    rows = [int(n) for n in rng.integers(0, 6, 75)]
    lens[3], lens[70], lens[40], lens[74] = 2500, 3100, 0, 1
    rows[3], rows[70], rows[40], rows[41], rows[74] = 5, 1, 2, 0, 5
    s = Stored(kv4, rng, heads, d, 16, lens, rows)
    s.fill(rng)
    for dtype in ("f16", "f32"):
        q = queries(rng, s, nh, dtype)
        s.batch.reserve(s.cache, nh)
        assert s.batch.work is not None
        s.batch.work.fill_(0xff)
        for causal, window in ((True, 0), (True, 90), (False, 0)):
            want, tol = s.expect(q, nh, causal, window, 0.125, dtype)
            check(attend(s, q, nh, dtype, causal, window), want, tol, dtype, f"{causal} {window}:")


def test_no_sequence_holds_a_token(kv4):
    """Lengths of zero throughout where the plan shares: every row is zeros."""
    say("empty")
    rng = np.random.default_rng(22)
    table = torch.zeros(3, 4096, dtype=torch.int32, device="cuda")
    cache = kv4.alloc(1, 16, 2, 128)
    cache.data.fill_(0xff)
    b = kv4.Batch(table, torch.zeros(3, dtype=torch.int32, device="cuda"), rows=2)
    assert b.reserve(cache, 4) > 0
    q = torch.from_numpy(rng.standard_normal((6, 4 * 128), dtype=np.float32)).cuda()
    out = torch.full_like(q, 5.0)
    for causal in (True, False):
        out.fill_(5)
        kv4.kvAttn(out, q, cache, b, 4, causal=causal)
        torch.cuda.synchronize()
        assert (out == 0).all()


def test_rows_cut_off_keep_their_positions(kv4):
    """Row r of a sequence is position len - rows_i + r also where m or `rows`
    leaves out the sequence's last rows: store, load and attention."""
    say("cut off")
    rng = np.random.default_rng(23)
    heads, d, page, lens, rows = 2, 64, 16, [40, 37, 30], [6, 9, 7]
    s = Stored(kv4, rng, heads, d, page, lens, rows)
    s.fill(rng)
    q = queries(rng, s, 4, "f32")
    want, tol = s.expect(q, 4, True, 0, 0.125, "f32")
    for m, most, kept in ((18, 9, list(range(18))), (22, 7, [*range(13), *range(15, 22)]), (3, 9, [0, 1, 2]), (0, 9, [])):
        b = kv4.Batch(s.batch.table, s.batch.lens, rows=most, row_off=s.batch.row_off, m=m)
        tq = torch.from_numpy(q.reshape(s.m, -1)).cuda()
        out = torch.full_like(tq, 9.0)
        kv4.kvAttn(out[:m], tq[:m], s.cache, b, 4)
        k, v = torch.full((2, s.m, heads * d), 9.0, device="cuda")
        kv4.kvLoad(s.cache, b, k[:m], v[:m])
        torch.cuda.synchronize()
        got, k = out.cpu().numpy().reshape(s.m, 4, d), k.cpu().numpy().reshape(s.m, heads, d)
        left = [r for r in range(s.m) if r not in kept]
        assert (got[left] == 9).all() and (k[left] == 9).all()
        if kept:
            check(got[kept].astype(np.float64), want[kept], tol[kept], "f32", f"m {m} rows {most}:")
        for i, n in enumerate(lens):
            for r, pos in enumerate(R.rows_of(n, rows[i])):
                if s.off[i] + r in kept:
                    kq, ks = s.held[i][:2]
                    assert np.array_equal(k[s.off[i] + r], R.value(kq[pos], ks[pos]).astype(np.float32))
        # a store through the same batch: the rows kept change, nothing else
        before = s.dev.clone()
        x = torch.from_numpy(rng.standard_normal((s.m, 2, heads * d), dtype=np.float32)).cuda()
        kv4.kvStore(s.cache, b, x[:m, 0], x[:m, 1])
        k, v = torch.empty(2, s.m, heads * d, device="cuda")
        kv4.kvLoad(s.cache, s.batch, k, v)
        torch.cuda.synchronize()
        for i, n in enumerate(lens):
            for r, pos in enumerate(R.rows_of(n, rows[i])):
                row = s.off[i] + r
                kq, ks = (R.quantise(x[row, 0].cpu().numpy().reshape(heads, d)) if row in kept
                          else (s.held[i][0][pos], s.held[i][1][pos]))
                assert np.array_equal(k[row].cpu().numpy().reshape(heads, d), R.value(kq, ks).astype(np.float32))
        s.dev.copy_(before)


def test_sequences_that_share_pages(kv4):
    """Three sequences with a common prefix in the same pages, one of them twice
    in the batch: what each would get alone, bit for bit between the twins."""
    say("shared pages")
    rng = np.random.default_rng(24)
    s = Stored(kv4, rng, 2, 128, 32, [96 + 20, 96 + 31, 96 + 20], [2, 2, 2])
    s.table[1, :3] = s.table[0, :3]
    s.table[2] = s.table[0]
    s.batch.table.copy_(torch.from_numpy(s.table))
    b = kv4.Batch(s.batch.table, s.batch.lens, rows=127, row_off=torch.tensor([0, 116, 243, 359], dtype=torch.int32).cuda(),
                  m=359)
    # stored one by one: the prefix once, then each one's own tokens
    x = rng.standard_normal((127 + 20, 2, 2, 128), dtype=np.float32).astype(np.float16)
    kv = torch.from_numpy(x).cuda()
    for i, n, lo, hi in ((1, 127, 0, 127), (0, 116, 127, 147)):
        one = kv4.Batch(s.batch.table[i:i + 1], s.batch.lens[i:i + 1], rows=hi - lo)
        kv4.kvStore(s.cache, one, kv[lo:hi, 0], kv[lo:hi, 1])
    torch.cuda.synchronize()
    prefix, own1, own0 = x[:96], x[96:127], x[127:]
    s.held = []
    for own in (own0, own1, own0):
        y = np.concatenate([prefix, own])
        s.held.append((*R.quantise(y[:, 0]), *R.quantise(y[:, 1]), np.ones(len(y), bool)))
    q = queries(rng, s, 8, "f16")
    q[4:] = q[:2]
    want, tol = s.expect(q, 8, True, 0, 128 ** -0.5, "f16")
    got = attend(s, q, 8, "f16")
    check(got, want, tol, "f16")
    assert np.array_equal(got[4:], got[:2])
    k, v = torch.empty(2, 359, 256, dtype=torch.float16, device="cuda")
    kv4.kvLoad(s.cache, b, k, v)
    torch.cuda.synchronize()
    assert torch.equal(k[:96], k[116:212]) and torch.equal(v[:116], v[243:])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_large_queries(kv4, dtype):
    """Rows up to the largest numbers of their type, and of the smallest."""
    say(f"large queries {dtype}")
    rng = np.random.default_rng(25)
    s = Stored(kv4, rng, 1, 64, 16, [200], [4])
    s.fill(rng)
    for top, scale in ((3e38, 2e-38), (1e36, 1e-36), (1e-36, 1e36)) if dtype == "f32" else ((65504.0, 1e-5), (2.0 ** -14, 1e4)):
        q = rng.uniform(-1, 1, (s.m, 2, 64))
        q[..., 0] = 1
        q = (q * top).astype(NP[dtype])
        want, tol = s.expect(q, 2, True, 0, float(np.float32(scale)), dtype)
        got = attend(s, q, 2, dtype, scale=scale)
        assert np.all(np.abs(got - want) <= tol), (top, (np.abs(got - want) / tol).max())


def test_two_streams_and_two_graphs_at_once(kv4):
    """Shared steps and their join on two streams at the same time, a workspace
    each: eagerly, then as captured graphs that are replayed several times with
    eager work between, lengths growing in place."""
    from madi_amd import q8
    say("two at once")
    rng = np.random.default_rng(26)
    heads, d, nh = 2, 128, 8
    s = Stored(kv4, rng, heads, d, 64, [9000, 5000], [1, 1])
    s.fill(rng)
    s.batch.lens.copy_(torch.tensor([8990, 4990], dtype=torch.int32))
    batches = [kv4.Batch(s.batch.table, s.batch.lens, rows=1) for _ in range(2)]
    for b in batches:
        assert b.reserve(s.cache, nh) > 0
    qs = [torch.from_numpy(rng.standard_normal((2, nh * d), dtype=np.float32)).cuda() for _ in range(2)]
    outs = [torch.zeros_like(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    held = s.held

    def expect(q, lens):
        s.lens = lens
        s.held = [tuple(a[:n] for a in h) for h, n in zip(held, lens)]
        return s.expect(q.cpu().numpy().reshape(2, nh, d), nh, True, 0, 128 ** -0.5, "f32")

    def right(lens, what):
        for o, q in zip(outs, qs):
            want, tol = expect(q, lens)
            check(o.cpu().numpy().reshape(2, nh, d).astype(np.float64), want, tol, "f32", what)

    torch.cuda.synchronize()
    try:
        for _ in range(4):  # in turn from the host, side by side on the device
            for st, b, q, o in zip(streams, batches, qs, outs):
                with torch.cuda.stream(st):
                    q8.init(st)
                    kv4.kvAttn(o, q, s.cache, b, nh)
        torch.cuda.synchronize()
        right([8990, 4990], "streams:")
        graphs = []
        for st, b, q, o in zip(streams, batches, qs, outs):
            g = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=st):
                q8.init(st)
                kv4.kvAttn(o, q, s.cache, b, nh)
            graphs.append(g)
        torch.cuda.synchronize()
        q8.init()
        for stepno in range(5):
            lens = [8991 + stepno, 4991 + stepno]
            s.batch.lens.copy_(torch.tensor(lens, dtype=torch.int32))
            for o in outs:
                o.fill_(3)
            torch.cuda.synchronize()
            for st, g in zip(streams, graphs):
                with torch.cuda.stream(st):
                    g.replay()
            torch.cuda.synchronize()
            eager = torch.empty_like(outs[0])
            kv4.kvAttn(eager, qs[0], s.cache, batches[0], nh)
            torch.cuda.synchronize()
            assert torch.equal(eager, outs[0])
            if stepno in (0, 4):
                right(lens, f"graphs {stepno}:")
    finally:
        torch.cuda.synchronize()
        q8.init()


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_large_scales_past_the_end(kv4, d, dtype):
    """The pool's other scales are the largest finite f16 numbers: what a
    sequence does not hold has no part in the exponent that its V scales share
    (with it, P would lose up to 16 bits), wherever in four tokens it ends."""
    say(f"large scales past the end {d} {dtype}")
    rng = np.random.default_rng(27)
    s = Setup(kv4, rng, 2, d, 16, [1, 18, 31, 44, 61], [1] * 5)
    s.data[..., 0::2], s.data[..., 1::2] = 0xff, 0x7b
    s.fill(rng)
    q = queries(rng, s, 4, dtype)
    want, tol = s.expect(q, 4, True, 0, d ** -0.5, dtype)
    got = attend(s, q, 4, dtype)
    for i in range(5):
        # (each row's own error: a single sequence's would be small beside the others)
        err = np.linalg.norm((got - want)[i]) / np.linalg.norm(want[i])
        assert err <= (5e-6 if dtype == "f32" else 2e-3), (i, err)
    check(got, want, tol, dtype)


@pytest.mark.parametrize("heads,group,d,lens,rows,window", [
    (2, 2, 64, [60, 37], [9, 5], 0), (1, 4, 128, [90, 133], [20, 40], 24), (2, 1, 96, [2500, 40], [3, 2], 0),
    (1, 2, 256, [50, 17], [16, 3], 8), (16, 16, 64, [230, 233], [230, 190], 40), (16, 16, 128, [250, 230], [230, 230], 0),
])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_infinities_that_a_row_does_not_see(kv4, heads, group, d, lens, rows, window, dtype):
    """K and V of each sequence's last token, and of one that all windows have
    passed, hold infinities and NaN: rows that do not see them lose nothing."""
    say(f"infinities {heads}x{group}x{d} {lens} {rows} window {window} {dtype}")
    rng = np.random.default_rng(28)
    s = Stored(kv4, rng, heads, d, 16, lens, rows)
    s.fill(rng)
    spots = [(i, n - 1) for i, n in enumerate(lens)]
    if window:
        spots += [(i, n - rows[i] - window) for i, n in enumerate(lens) if n - rows[i] - window >= 0]
    for i, pos in spots:
        x = rng.standard_normal((1, 2, heads, d)).astype(np.float32)
        x[..., ::5], x[..., 1::7], x[..., 2::9] = np.inf, -np.inf, np.nan
        one = kv4.Batch(s.batch.table[i:i + 1], torch.tensor([pos + 1], dtype=torch.int32).cuda(), rows=1)
        kv = torch.from_numpy(x).cuda()
        kv4.kvStore(s.cache, one, kv[:, 0], kv[:, 1])
        torch.cuda.synchronize()
        for held, new in zip(s.held[i], (*R.quantise(x[:, 0]), *R.quantise(x[:, 1]))):
            held[pos] = new[0]
    nh = heads * group
    q = queries(rng, s, nh, dtype)
    want, tol = s.expect(q, nh, True, window, d ** -0.5, dtype)
    got = attend(s, q, nh, dtype, True, window)
    unseen = [s.off[i] + r for i, n in enumerate(lens) for r, pos in enumerate(R.rows_of(n, rows[i])) if pos < n - 1]
    err = np.linalg.norm((got - want)[unseen], axis=-1) / np.maximum(np.linalg.norm(want[unseen], axis=-1), 1e-3)
    say(f"  worst row {err.max():.2e}")
    # (a row's own error: for f32 rows its scores' and the 22 bits of q and P, for f16 rows two roundings)
    assert err.max() <= (2e-5 if dtype == "f32" else 2e-3)
    seen = [r for r in range(s.m) if r not in unseen]
    assert np.all(np.abs(got - want)[seen] <= tol[seen])


@pytest.mark.parametrize("heads,group,d,lens,rows", [
    (2, 4, 64, [5000, 40], [3, 3]), (16, 16, 64, [230, 233], [230, 190]), (1, 20, 128, [300, 9], [4, 2])])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_in_place_on_every_path(kv4, heads, group, d, lens, rows, dtype):
    """out = q where steps are shared and joined, in the prompts' kernel, and with
    more columns than a tile; then with a hint far below the lengths."""
    say(f"in place {heads}x{group}x{d} {lens} {rows} {dtype}")
    rng = np.random.default_rng(29)
    s = Stored(kv4, rng, heads, d, 16, lens, rows)
    s.fill(rng)
    nh = heads * group
    q = queries(rng, s, nh, dtype)
    want, tol = s.expect(q, nh, True, 0, d ** -0.5, dtype)
    s.batch.reserve(s.cache, nh)
    tq = torch.from_numpy(q.reshape(s.m, -1)).cuda()
    s.kv4.kvAttn(tq, tq, s.cache, s.batch, nh)
    torch.cuda.synchronize()
    check(tq.cpu().numpy().reshape(q.shape).astype(np.float64), want, tol, dtype, "in place:")
    b = kv4.Batch(s.batch.table, s.batch.lens, rows=max(rows), row_off=s.batch.row_off, m=s.m, len_max=5)
    tq = torch.from_numpy(q.reshape(s.m, -1)).cuda()
    out = torch.empty_like(tq)
    s.kv4.kvAttn(out, tq, s.cache, b, nh)
    torch.cuda.synchronize()
    check(out.cpu().numpy().reshape(q.shape).astype(np.float64), want, tol, dtype, "hint:")
