"""Attention over the 4-bit cache with V of every magnitude: the power of two that a
column's V scales share follows them as they grow along a sequence, differs between
the waves and segments that are joined, and has to leave small V their bits.

Tolerance: test_gpu_kv4.py's, with one term in place of 2^-32 sum|v|: a weight times its
V scale lies on f16's finest grid, 2^-24 of 2^e <= 2 s, s the largest V scale of the
head, where the largest weight is at least 2^7 2^-e.  Each key's 7 codes are off by half of
that, n keys' outputs by n * 7 * 2^-25 * 2 s / 2^7 = 7 n s 2^-31.  Long prompts hold V itself
as two f16; products of V below 2^-14 add up to 2^-18 of their sum of magnitudes, and the
grid is the weights' alone, 2^-25 / 2^7 of |v| (2^-32 sum|v|, which 7 n s 2^-31 is above)."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import NP, Setup, attend, check, kv4, say  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

PATHS = [
    # heads, group, d, page, lens, rows, causal, window, long prompts
    (2, 2, 64, 16, [200, 33, 1], [1, 3, 1], True, 0, False),
    (1, 4, 96, 32, [300, 90], [2, 20], True, 40, False),
    (2, 5, 256, 16, [150, 41], [2, 1], False, 0, False),
    (2, 4, 64, 64, [5000, 40], [1, 3], True, 0, False),        # steps shared by workgroups
    (1, 8, 128, 16, [4100, 2222], [1, 1], True, 3000, False),
    (1, 2, 256, 128, [2500], [1], True, 0, False),
    (4, 64, 64, 16, [230, 233], [230, 233], True, 0, True),
    (4, 64, 128, 16, [230, 233], [230, 233], True, 0, True),
]


def magnitudes(kind, n):
    t = np.arange(n) / max(n - 1, 1)
    if kind == "small":
        return np.full(n, 3e-6)
    if kind == "zero":
        return np.zeros(n)
    if kind == "zero first":
        return np.where(t < 0.6, 0, 5.0)
    if kind == "growing":
        return 10.0 ** (-5 + 8 * t)
    if kind == "falling":
        return 10.0 ** (3 - 8 * t)
    return np.where(np.arange(n) % 7 == 3, 8000.0, 1e-3)  # "mixed"


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("kind,heads,group,d,page,lens,rows,causal,window,prompt",
                         [(k, *p) for p in PATHS for k in ("small", "zero", "zero first", "growing", "falling", "mixed")
                          if not p[-1] or k in ("small", "zero first", "mixed")])
def test_values_of_every_magnitude(kv4, kind, heads, group, d, page, lens, rows, causal, window, prompt, dtype):
    say(f"V {kind} {heads}x{group}x{d} {lens} {rows} {dtype}")
    rng = np.random.default_rng(sum(lens) + d)
    s = Setup(kv4, rng, heads, d, page, lens, rows)
    s.fill(rng)
    for i, n in enumerate(lens):
        kq, ks, vq, vs, there = s.held[i]
        v = rng.standard_normal((n, heads, d)) * magnitudes(kind, n)[:, None, None]
        vq[:], vs[:] = R.quantise(v.astype(np.float32))
        for t in range(n):
            p, o = s.place(i, t)
            for h in range(heads):
                R.put(s.data, page, d, p, h, o, kq[t, h], ks[t, h], vq[t, h], vs[t, h])
    s.dev.copy_(torch.from_numpy(s.data))
    nh = heads * group
    q = rng.standard_normal((s.m, nh, d), dtype=np.float32).astype(NP[dtype])
    want, tol = np.zeros((s.m, nh, d)), np.zeros((s.m, nh, d))
    for i, n in enumerate(lens):
        kq, ks, vq, vs, there = s.held[i]
        r0, r1 = s.off[i], s.off[i + 1]
        for h in range(heads):
            c = slice(h * group, (h + 1) * group)
            o, a, _ = R.attention(q[r0:r1, c], R.value(kq[:, h], ks[:, h]), R.value(vq[:, h], vs[:, h]), there,
                                  list(R.rows_of(n, r1 - r0)), causal, window, d ** -0.5)
            e = R.score_error(q[r0:r1, c], ks[:, h], d ** -0.5)[..., None]
            unit = 2.0 ** -10 if dtype == "f16" else 3 * 2.0 ** -22
            if prompt:
                unit += 2.0 ** -18
            last = 2.0 ** -11 * np.abs(o) + 2.0 ** -25 if dtype == "f16" else 2.0 ** -24 * np.abs(o)
            want[r0:r1, c] = o
            tol[r0:r1, c] = ((unit + 2 * e + 32 * 2.0 ** -23 + (n / 32 + 64) * 2.0 ** -24) * a + last +
                             7 * n * float(vs[:, h].astype(np.float64).max(initial=0)) * 2.0 ** -31)
    got = attend(s, q, nh, dtype, causal, window)
    assert np.all(np.isfinite(got))
    assert kind != "zero" or not got.any()
    worst = (np.abs(got - want) / np.maximum(tol, 1e-300)).max()
    norm = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
    say(f"  worst |err| / tol {worst:.3f}, normwise {norm:.2e}")
    assert worst <= 1
    if s.batch.work is not None:
        s.batch._c.work, s.batch._c.work_bytes = None, 0
        alone = attend(s, q, nh, dtype, causal, window, reserve=False)
        assert np.all(np.abs(alone - want) <= tol)
