"""The 4-bit cache without a GPU: sizes, refusals before a device is touched,
the Python wrappers' checks, and the reference's own arithmetic."""
import ctypes

import numpy as np
import pytest

import kv4_ref as R
import madi_amd
from madi_amd import _lib, kv4

torch = pytest.importorskip("torch")

FAKE = 0x100000  # 16-byte aligned, never dereferenced
FAR = 0x40000000


def cache(data=FAKE, n_pages=4, page=16, nkv=2, d=64):
    return kv4._Cache(data, n_pages, page, nkv, d)


def batch(table=FAR, lens=FAR, row_off=None, b=2, max_pages=2, rows=3, m=6, len_max=0, work=None, work_bytes=0):
    return kv4._Batch(table, lens, row_off, b, max_pages, rows, m, len_max, work, work_bytes)


def call(name, *args):
    return getattr(madi_amd.lib(), name)(*[ctypes.addressof(a) if isinstance(a, ctypes.Structure) else a
                                           for a in args])


def test_sizes():
    b = madi_amd.lib().madi_kv4_bytes
    assert b(3, 16, 2, 64) == 3 * 2 * R.block_bytes(16, 64)
    assert b(1 << 20, 1024, 8, 128) == (1 << 20) * 8 * R.block_bytes(1024, 128)  # past 32 bits
    for bad in ((1, 15, 1, 64), (1, 24, 1, 64), (1, 8, 1, 64), (1, 16, 0, 64), (1, 16, 1, 80), (1, 16, 1, 512),
                (1, 1 << 25, 1, 64), (1, 16, 65536, 64)):
        assert b(*bad) == 0, bad
    assert ctypes.sizeof(kv4._Cache) == 24 and ctypes.sizeof(kv4._Batch) == 64


SHAPES = [
    (cache(page=24), batch(), -5), (cache(d=80), batch(), -5), (cache(nkv=0), batch(), -5),
    (cache(n_pages=0), batch(), -5), (cache(), batch(m=5), -5), (cache(), batch(b=65536, m=3 * 65536), -5),
    (cache(), batch(max_pages=0), -5), (cache(), batch(max_pages=1 << 27), -5),
    (cache(), batch(rows=1 << 31, row_off=FAR), -5), (cache(), batch(m=1 << 31, row_off=FAR), -5),
    (cache(data=None), batch(), -6), (cache(), batch(table=None), -6), (cache(), batch(lens=None), -6),
    (cache(data=FAKE + 8), batch(), -7), (cache(), batch(table=FAR + 2), -7), (cache(), batch(row_off=FAR + 1), -7),
    (cache(), batch(), -8), (cache(), batch(row_off=FAR, m=5), -8), (cache(), batch(b=0, m=0), -8),
]


@pytest.mark.parametrize("c,b,code", SHAPES)
def test_refusals_all_entry_points_share(c, b, code):
    k, v = FAR + 0x100000, FAR + 0x200000
    assert call("madi_kv4_store", c, b, k, v, 128, 128, 0) == code, _lib.last_error()
    assert call("madi_kv4_load", k, v, 128, 128, 0, c, b) == code
    assert call("madi_kv4_attn", k, v, c, b, 4, 256, 256, 0, 1, 0, 0.125) == code
    assert _lib.last_error()


def test_refusals_of_structs_and_rows():
    c, b, k, v = cache(), batch(), FAR + 0x100000, FAR + 0x200000
    assert call("madi_kv4_store", None, b, k, v, 128, 128, 0) == -6
    assert call("madi_kv4_store", c, None, k, v, 128, 128, 0) == -6
    for f in (lambda k, v, lk, lv, dt: call("madi_kv4_store", c, b, k, v, lk, lv, dt),
              lambda k, v, lk, lv, dt: call("madi_kv4_load", k, v, lk, lv, dt, c, b)):
        assert f(k, v, 127, 128, 0) == -5       # rows longer than apart
        assert f(k, v, 128, 0, 0) == -5
        assert f(None, v, 128, 128, 0) == -6
        assert f(k, None, 128, 128, 0) == -6
        assert f(k + 8, v, 128, 128, 0) == -7
        assert f(k, v, 132, 128, 0) == -7       # 264 bytes
        assert f(k, v, 132, 128, 1) == -8       # 528 bytes
        assert f(k, v, 128, 130, 1) == -7
        assert f(k, v, 128, 128, 2) == -9
        assert f(FAKE, v, 128, 128, 0) == -9    # in the cache
        assert f(k, FAKE + 1024, 128, 128, 0) == -9
        assert f(k, k + 256, 256, 256, 0) == -8  # k | v alternate
    assert call("madi_kv4_load", k, k + 128, 128, 128, 0, c, b) == -9
    assert call("madi_kv4_load", k, k + 128, 256, 256, 0, c, b) == -9
    assert call("madi_kv4_load", k, k + 256 * 2, 256, 128, 0, c, b) == -9
    assert call("madi_kv4_store", c, b, k, k, 128, 128, 0) == -8   # K and V may be one


@pytest.mark.parametrize("args,code", [
    (dict(nh=3), -5), (dict(nh=0), -5), (dict(ldq=255), -5), (dict(ldo=128), -5), (dict(q=None), -6),
    (dict(out=None), -6), (dict(q=FAR + 0x200002), -7), (dict(ldo=260), -7), (dict(causal=2), -9),
    (dict(causal=0, window=5), -9), (dict(dtype=7), -9), (dict(scale=float("nan")), -9),
    (dict(scale=float("inf")), -9), (dict(out=FAKE + 16), -9), (dict(out=FAR + 0x200000 + 512), -9),
    (dict(out=FAR + 0x200000), -8), (dict(out=FAR + 0x200000, ldo=512), -9), (dict(window=0xffffffff), -8),
    (dict(work=FAR + 0x100008, work_bytes=1 << 20), -7), (dict(work=FAR + 0x100000, work_bytes=64), -9),
    (dict(work=FAR + 0x200000, work_bytes=64), -9), (dict(work=FAKE, work_bytes=64), -9),
    (dict(work=FAR + 0x900000, work_bytes=64), -8), (dict(rows=1 << 30, row_off=FAR), -5), (dict(), -8),
])
def test_refusals_of_attention(args, code):
    a = dict(out=FAR + 0x100000, q=FAR + 0x200000, nh=4, ldo=256, ldq=256, window=0, causal=1, dtype=0, scale=0.125)
    b = batch(**{k: args.pop(k) for k in list(args) if k in ("work", "work_bytes", "rows", "row_off")})
    a.update(args)
    rc = call("madi_kv4_attn", a["out"], a["q"], cache(), b, a["nh"], a["ldo"], a["ldq"], a["window"], a["causal"],
              a["dtype"], a["scale"])
    assert rc == code, (rc, _lib.last_error())


def test_workspace_size():
    f = lambda c, b, nh: call("madi_kv4_attn_bytes", c, b, nh)
    assert f(cache(), batch(), 4) == 0                       # a short cache is not split
    long = batch(b=1, max_pages=8192, rows=1, m=1)
    assert 0 < f(cache(), long, 4) < 64 << 20
    assert f(cache(), batch(b=1, max_pages=8192, rows=1, m=1, len_max=100), 4) == 0
    assert f(cache(), long, 3) == 0 and f(cache(d=80), long, 4) == 0


def test_wrappers_refuse():
    data = torch.zeros(4 * 2 * R.block_bytes(16, 64), dtype=torch.uint8)
    c = kv4.KV4(data, page=16, heads=2, dim=64)
    assert c.n_pages == 4
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    b = kv4.Batch(table, lens, rows=3)
    k = torch.zeros(6, 128)
    bad = [lambda: kv4.KV4(data, page=16, heads=2, dim=80), lambda: kv4.KV4(data, page=16, heads=2, dim=64, n_pages=5),
           lambda: kv4.KV4(data[::2], page=16, heads=2, dim=64), lambda: kv4.alloc(1, 17, 2, 64, device="cpu"),
           lambda: kv4.alloc(-1, 16, 2, 64, device="cpu"),
           lambda: kv4.Batch(table[0], lens), lambda: kv4.Batch(table, lens[:1]),
           lambda: kv4.Batch(table.float(), lens), lambda: kv4.Batch(table.long(), lens),
           lambda: kv4.Batch(table, lens, rows=-1), lambda: kv4.Batch(table, lens, row_off=lens, m=3),
           lambda: kv4.Batch(table, lens, row_off=torch.zeros(3, dtype=torch.int32)),
           lambda: kv4.Batch(table.T, lens), lambda: kv4.Batch(table, lens, rows=3, m=5) and kv4.kvStore(
               c, kv4.Batch(table, lens, rows=3, m=5), k, k),
           lambda: kv4.kvStore(c, b, k[:5], k), lambda: kv4.kvStore(c, b, k.double(), k.double()),
           lambda: kv4.kvStore(c, b, k, k.half()), lambda: kv4.kvStore(c, b, k.T, k),
           lambda: kv4.kvStore(c, b, k[:, :64], k), lambda: kv4.kvLoad(c, b, k, k.half()),
           lambda: kv4.kvStore(c, b, torch.zeros(1, 128).expand(6, 128), k),
           lambda: kv4.kvStore(c, b, torch.zeros(6, 2, 128)[:, :, ::2], k),
           lambda: kv4.kvAttn(k, k, c, b, nh=4), lambda: kv4.kvAttn(k, k.half(), c, b, nh=2),
           lambda: kv4.kvAttn(k, k.clone(), c, b, nh=2, causal=False, window=3)]
    for f in bad:
        with pytest.raises(madi_amd.MadiError):
            f()
    for f in (lambda: kv4.kvStore(c, b, k, k.view(6, 2, 64)), lambda: kv4.kvAttn(k, k, c, b, nh=2)):
        with pytest.raises(madi_amd.MadiError) as e:
            f()
        assert e.value.code == -8  # accepted up to the device


def test_the_format():
    """The definition on its own terms: a code's value is the nearest one (ties
    away from zero), infinities and NaN as stated, the block maximum 7 s."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((200, 64)).astype(np.float32) * 10.0 ** rng.integers(-6, 5, (200, 1))
    x = x.astype(np.float32)
    q, s = R.quantise(x)
    v = R.value(q, s)
    step = s.astype(np.float64).repeat(32, -1)
    # half a step, plus what the scale's rounding takes from 7 s: 2^-11 of 7 s for a
    # normal f16 s, 7 * 2^-25 for a subnormal one
    tol = step * (0.5 + 2.0 ** -7) + 7 * 2.0 ** -25
    assert np.all(np.abs(v - x) <= np.where(s.repeat(32, -1) < 9352, tol, np.inf))
    assert np.all(np.abs(q) <= 7) and np.all(np.isfinite(v)) and np.abs(v).max() <= 65464
    y = np.zeros(64, np.float32)
    y[0], y[1], y[2], y[3] = np.inf, -np.inf, np.nan, 1e5
    q, s = R.quantise(y)
    assert list(s) == [9352, 0] and list(q[:4]) == [7, -7, 0, 7] and not q[4:].any()
    y = np.float32([7, 0.5, -0.5, 1.5, 0.49999997, -2.5] + [0] * 26)
    assert list(R.quantise(y)[0][:6]) == [7, 1, -1, 2, 0, -3]


def test_sizes_past_what_an_address_or_a_launch_holds():
    """Pages of more than 2^20 tokens, caches past 2^48 bytes (their product
    would wrap) and launches of 2^32 threads are refused."""
    b = madi_amd.lib().madi_kv4_bytes
    assert b(1, 1 << 20, 1, 256) == 288 << 20
    assert b(1, 1 << 21, 1, 64) == 0
    assert b(0xffffffff, 1 << 20, 65535, 256) == 0 and b(0xffffffff, 16, 1, 64) == 0xffffffff * 16 * 72
    k, v = FAR + 0x100000, FAR + 0x200000
    for c in (cache(page=1 << 21), cache(n_pages=0xffffffff, page=1 << 20, nkv=2)):
        assert call("madi_kv4_store", c, batch(), k, v, 128, 128, 0) == -5
        assert call("madi_kv4_attn", k, v, c, batch(), 4, 256, 256, 0, 1, 0, 0.125) == -5
    many = batch(row_off=FAR, rows=0x7fffffff)
    assert call("madi_kv4_store", cache(nkv=256), many, k, v, 1 << 14, 1 << 14, 0) == -5
    assert call("madi_kv4_attn", k, v, cache(), many, 4, 256, 256, 0, 1, 0, 0.125) == -5
    with pytest.raises(madi_amd.MadiError):
        kv4._bytes(0xffffffff, 1 << 20, 65535, 256)


def test_the_workspace_serves_every_type_and_window():
    """What a batch reserves does not depend on which kernel f16 rows without a
    window would take: prompts with a window may be split too."""
    f = lambda b: call("madi_kv4_attn_bytes", cache(nkv=8, d=128), b, 32)
    one = f(batch(b=1, max_pages=8192, rows=1, m=1))
    assert f(batch(b=1, max_pages=8192, rows=2048, m=2048)) >= one > 0


def test_a_call_without_rows():
    """No rows: no row pointers are needed (torch gives an empty tensor none)."""
    b = batch(b=0, m=0)
    assert call("madi_kv4_store", cache(), b, None, None, 128, 128, 0) == -8  # (madi_init, as for any other call)
    assert call("madi_kv4_attn", None, None, cache(), b, 4, 256, 256, 0, 1, 0, 0.125) == -8


def test_wrappers_refuse_what_32_bits_do_not_hold():
    """Distances and windows past 32 bits would wrap to other, valid ones."""
    c = kv4.KV4(torch.zeros(4 * 2 * R.block_bytes(16, 64), dtype=torch.uint8), page=16, heads=2, dim=64)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    b, one = kv4.Batch(table, lens, rows=2), kv4.Batch(table, lens, rows=1)
    far = torch.empty_strided((2, 128), ((1 << 32) + 128, 1), dtype=torch.float16, device="meta")
    near = torch.zeros(2, 128, dtype=torch.float16)
    for f in (lambda: kv4.kvStore(c, b, far, far), lambda: kv4.kvLoad(c, b, near, far),
              lambda: kv4.kvAttn(far, near, c, b, nh=2), lambda: kv4.kvAttn(near, near, c, b, nh=2, window=(1 << 32) + 5),
              lambda: kv4.kvAttn(near, near, c, b, nh=2, window=-1)):
        with pytest.raises(madi_amd.MadiError) as e:
            f()
        assert e.value.code == -5
    # a single row is not apart from any other
    for k in (torch.empty_strided((1, 128), ((1 << 32) + 128, 1), dtype=torch.float16, device="meta"),):
        with pytest.raises(madi_amd.MadiError) as e:
            kv4.kvStore(c, one, k, near[:1])
        assert e.value.code == -6  # (a meta tensor has no address)


@pytest.mark.parametrize("d,whole", [(64, 2048), (96, 2048), (128, 1024), (256, 1024)])
def test_the_workspace_serves_both_types_at_every_length(d, whole):
    """Rows of one type are split from shorter caches on than the other's (d = 128: f32
    from 1025 keys, f16 from 2049): there is a workspace wherever either is."""
    f = lambda n: call("madi_kv4_attn_bytes", cache(nkv=8, d=d), batch(b=1, max_pages=8192, rows=1, m=1, len_max=n), 32)
    assert f(whole) == 0
    for n in (whole + 1, 1500, 2048, 2049, 4096, 131072):
        assert (f(n) > 0) == (n > whole), n
    sizes = [f(n) for n in (2049, 4096, 131072)]
    assert min(sizes) == max(sizes)


@pytest.mark.parametrize("what,size", [("table", 16), ("lens", 8), ("row_off", 12)])
def test_what_a_call_reads_is_not_written_by_it(what, size):
    """table, lens and row_off under out, work, k, v or the cache are refused, beside
    them taken; under what a call only reads too."""
    c, x, y = cache(), FAR + 0x100000, FAR + 0x200000
    work = dict(work=FAR + 0x900000, work_bytes=512)
    rows, attn, held = (5 * 256 + 128) * 2, 6 * 256 * 2, 4 * 2 * R.block_bytes(16, 64)
    writes = [
        (x, rows, lambda b: call("madi_kv4_load", x, y, 256, 256, 0, c, b)),
        (y, rows, lambda b: call("madi_kv4_load", x, y, 256, 256, 0, c, b)),
        (x, attn, lambda b: call("madi_kv4_attn", x, y, c, b, 4, 256, 256, 0, 1, 0, 0.125)),
        (work["work"], 512, lambda b: call("madi_kv4_attn", x, y, c, b, 4, 256, 256, 0, 1, 0, 0.125)),
        (FAKE, held, lambda b: call("madi_kv4_store", c, b, x, y, 256, 256, 0)),
    ]
    for start, length, f in writes:
        for at, code in ((start - size, -8), (start - size + 4, -9), (start, -9), (start + length - 4, -9),
                         (start + length, -8)):
            assert f(batch(**{"row_off": FAR, **work, what: at})) == code, (hex(at), _lib.last_error())
    for at in (x, y):
        assert call("madi_kv4_store", c, batch(**{"row_off": FAR, what: at}), x, y, 256, 256, 0) == -8
    assert call("madi_kv4_attn", x, y, c, batch(**{"row_off": FAR, what: y}), 4, 256, 256, 0, 1, 0, 0.125) == -8
    # (of one token: no row starts are read without row_off)
    assert call("madi_kv4_attn", x, y, c, batch(), 4, 256, 256, 0, 1, 0, 0.125) == -8


def test_positions_end_before_31_bits_do():
    """A step of keys that begins below 2^31 would end past it: the last 4096 positions
    are refused."""
    k, v = FAR + 0x100000, FAR + 0x200000
    for page, most in ((16, (1 << 31) - 4096), (4096, (1 << 31) - 4096), (1 << 20, (1 << 31) - (1 << 20))):
        c = cache(page=page)
        for pages, code in ((most // page, -8), (most // page + 1, -5)):
            b = batch(max_pages=pages, table=FAR + (1 << 32))
            assert call("madi_kv4_store", c, b, k, v, 128, 128, 0) == code
            assert call("madi_kv4_load", k, v, 128, 128, 0, c, b) == code
            assert call("madi_kv4_attn", k, v, c, b, 4, 256, 256, 0, 1, 0, 0.125) == code
