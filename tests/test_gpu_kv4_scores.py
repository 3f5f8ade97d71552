"""Attention over the 4-bit cache where scores are large: f32 numbers of 10^8 and
more lie further apart than the softmax's references are from the largest
score, and beyond 10^30 (below -10^30) there are scores as well.  Tolerances:
test_gpu_kv4.py's without the score's error, for the rows where that cannot
matter: the largest score is ahead of the others by more than twice its bound and 64
more (e^-64 of the others' |V| is below every other term), or the keys are
all alike, so that the same roundings give them the same score."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import NP, Setup, check, kv4, say  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

PATHS = [
    # heads, group, d, page, lens, rows, causal: lengths of one among them
    (2, 2, 64, 16, [1, 200, 1, 70], [1] * 4, True),              # a workgroup per tile and head
    (1, 4, 128, 16, [1, 300, 33], [1, 5, 2], True),
    (2, 4, 96, 64, [1, 3000, 1, 2300], [1, 2, 1, 1], True),      # steps shared by workgroups
    (1, 2, 256, 16, [2100, 1], [1, 1], True),
    (4, 64, 64, 16, [230, 233], [230, 233], True),              # the prompts' kernel
    (4, 64, 128, 16, [230, 233], [230, 233], True),
]


def rows_of_one_key(s, q, nh, causal, scale):
    """Per row and head whether one key decides alone, by the score's bound."""
    g, alone = nh // s.heads, np.zeros((s.m, nh), bool)
    for i, n in enumerate(s.lens):
        kq, ks = s.held[i][:2]
        r0, r1 = s.off[i], s.off[i + 1]
        pos = np.array(R.rows_of(n, r1 - r0))[:, None]
        for h in range(s.heads):
            qh = q[r0:r1, h * g:(h + 1) * g].astype(np.float64)
            k = R.value(kq[:, h], ks[:, h])
            x = (qh.reshape(-1, s.d) @ k.T).reshape(r1 - r0, g, n) * scale
            if causal:
                x = np.where((np.arange(n)[None] <= pos)[:, None], x, -np.inf)
            x = np.sort(x, -1)
            bound = R.score_error(qh, ks[:, h], scale)
            alone[r0:r1, h * g:(h + 1) * g] = (x[..., -1] - x[..., -2] > 2 * bound + 64) if n > 1 else True
    return alone


def one_key_outputs(s, q, nh, causal, dtype, scale=None):
    """Exact outputs, and the bound of test_gpu_kv4.py where one key's V is the output and
    scores have no error: the mean |v| is the output's own."""
    want, _ = s.expect(q, nh, causal, 0, scale or s.d ** -0.5, dtype)
    n = np.repeat([max(n, 1) for n in s.lens], np.diff(s.off))[:, None, None]
    unit = 2.0 ** -10 + 2.0 ** -11 if dtype == "f16" else 3 * 2.0 ** -22 + 2.0 ** -24
    tol = (unit + 32 * 2.0 ** -23 + (n / 32 + 64) * 2.0 ** -24) * np.abs(want)
    return want, tol + (2.0 ** -25 if dtype == "f16" else 0) + 1e-25  # (e^-64 of the others)


@pytest.mark.parametrize("dtype,top", [("f32", 1e7), ("f32", 3e8), ("f32", 1e10), ("f32", 1e34), ("f16", 300),
                                       ("f16", 6e4)])
@pytest.mark.parametrize("heads,group,d,page,lens,rows,causal", PATHS)
def test_large_scores(kv4, heads, group, d, page, lens, rows, causal, dtype, top):
    say(f"large scores {heads}x{group}x{d} {lens} {rows} {dtype} {top:g}")
    rng = np.random.default_rng(sum(lens) + d)
    s = Setup(kv4, rng, heads, d, page, lens, rows)
    s.fill(rng, spread=1.0 if dtype == "f32" else 1e4)
    nh = heads * group
    q = rng.uniform(-1, 1, (s.m, nh, d))
    q = (q * top).astype(NP[dtype])
    want, tol = one_key_outputs(s, q, nh, causal, dtype)
    alone = rows_of_one_key(s, q, nh, causal, d ** -0.5)
    assert alone.mean() > 0.5, alone.mean()
    tq = torch.from_numpy(q.reshape(s.m, -1)).cuda()
    for reserved in (True, False):
        if reserved:
            s.batch.reserve(s.cache, nh)
        else:
            s.batch._c.work, s.batch._c.work_bytes = None, 0
        out = torch.full_like(tq, 77.0)
        kv4.kvAttn(out, tq, s.cache, s.batch, nh, causal=causal)
        torch.cuda.synchronize()
        got = out.cpu().numpy().reshape(s.m, nh, d).astype(np.float64)
        assert np.all(np.isfinite(got))
        check(got[alone], want[alone], tol[alone], dtype, f"{alone.mean():.2f} of the rows:")
        # the others are means of V's rows, whatever the weights
        for i in range(len(lens)):
            v = R.value(s.held[i][2], s.held[i][3])
            lo, hi = (f(0).repeat(group, 0) for f in (v.min, v.max))
            slack = 2.0 ** -9 * np.maximum(np.abs(lo), np.abs(hi))
            o = got[s.off[i]:s.off[i + 1]]
            assert np.all(o >= lo - slack) and np.all(o <= hi + slack)


@pytest.mark.parametrize("dtype,top", [("f32", 1.0), ("f32", 3e8), ("f32", 1e10), ("f32", -1e32), ("f16", 6e4),
                                       ("f16", -6e4)])
@pytest.mark.parametrize("heads,group,d,page,lens,rows,causal", PATHS)
def test_keys_that_are_alike(kv4, heads, group, d, page, lens, rows, causal, dtype, top):
    """Every key the same, so every score: the mean of V, however large the score is,
    and of either sign."""
    say(f"alike {heads}x{group}x{d} {lens} {rows} {dtype} {top:g}")
    rng = np.random.default_rng(sum(lens) + d + 1)
    s = Setup(kv4, rng, heads, d, page, lens, rows)
    s.fill(rng)
    code = rng.integers(1, 8, d)
    scale = np.full(d // 32, 0.75 if dtype == "f32" else 3000, np.float16)
    for i, n in enumerate(lens):
        kq, ks, vq, vs, there = s.held[i]
        kq[:], ks[:] = code, scale
        for t in range(n):
            p, o = s.place(i, t)
            for h in range(heads):
                R.put(s.data, page, d, p, h, o, kq[t, h], ks[t, h], vq[t, h], vs[t, h])
    s.dev.copy_(torch.from_numpy(s.data))
    nh = heads * group
    q = (rng.uniform(0.5, 1, (s.m, nh, d)) * top).astype(NP[dtype])
    # the mean of V with equal weights, and of |V|
    want, tol = np.zeros((s.m, nh, d)), np.zeros((s.m, nh, d))
    for i, n in enumerate(lens):
        v = R.value(s.held[i][2], s.held[i][3])
        for r, pos in enumerate(R.rows_of(n, rows[i])):
            if pos < 0:
                continue
            k = pos + 1 if causal else n
            o, a, most = (x.repeat(group, 0) for x in (v[:k].mean(0), np.abs(v[:k]).mean(0), np.abs(v[:k]).sum(0)))
            unit = 2.0 ** -10 if dtype == "f16" else 3 * 2.0 ** -22
            last = 2.0 ** -11 if dtype == "f16" else 2.0 ** -24
            want[s.off[i] + r] = o
            tol[s.off[i] + r] = ((unit + 32 * 2.0 ** -23 + (n / 32 + 64) * 2.0 ** -24) * a + last * np.abs(o) +
                                 2.0 ** -32 * most + (2.0 ** -25 if dtype == "f16" else 0))
    tq = torch.from_numpy(q.reshape(s.m, -1)).cuda()
    out = torch.full_like(tq, 77.0)
    s.batch.reserve(s.cache, nh)
    kv4.kvAttn(out, tq, s.cache, s.batch, nh, causal=causal)
    torch.cuda.synchronize()
    check(out.cpu().numpy().reshape(s.m, nh, d).astype(np.float64), want, tol, dtype)


@pytest.mark.parametrize("top,scale", [(3e38, 2e-38), (1e36, 1e-36), (1e-36, 1e36)])
@pytest.mark.parametrize("heads,group,d,page,lens,rows", [(4, 64, 64, 16, [230, 233], [230, 233]),
                                                           (4, 64, 256, 16, [200, 217], [200, 217])])
def test_prompts_of_large_and_small_rows(kv4, heads, group, d, page, lens, rows, top, scale):
    """f32 rows up to the largest numbers and of the smallest, the scale bringing the scores back."""
    say(f"prompt rows of {top:g}, scale {scale:g}, d {d}")
    rng = np.random.default_rng(31)
    s = Setup(kv4, rng, heads, d, page, lens, rows)
    s.fill(rng, spread=0.01)
    nh = heads * group
    q = (rng.uniform(-1, 1, (s.m, nh, d)) * top).astype(np.float32)
    want, tol = s.expect(q, nh, True, 0, float(np.float32(scale)), "f32")
    tq = torch.from_numpy(q.reshape(s.m, -1)).cuda()
    out = torch.full_like(tq, 77.0)
    kv4.kvAttn(out, tq, s.cache, s.batch, nh, scale=scale)
    torch.cuda.synchronize()
    check(out.cpu().numpy().reshape(s.m, nh, d).astype(np.float64), want, tol, "f32")


@pytest.mark.parametrize("heads,group,d,page,lens,rows,causal", PATHS)
def test_rows_of_zeros_under_a_large_scale(kv4, heads, group, d, page, lens, rows, causal):
    """Rows of 10^-36 with a scale of 10^36, among them (padding) rows of zeros: the mean of V."""
    say(f"rows of zeros {heads}x{group}x{d} {lens}")
    rng = np.random.default_rng(sum(lens) + 5)
    s = Setup(kv4, rng, heads, d, page, lens, rows)
    s.fill(rng, spread=0.01)
    nh = heads * group
    q = (rng.uniform(-1, 1, (s.m, nh, d)) * 1e-36).astype(np.float32)
    q[rng.random((s.m, nh)) < 0.5] = 0
    want, tol = s.expect(q, nh, causal, 0, float(np.float32(1e36)), "f32")
    tq = torch.from_numpy(q.reshape(s.m, -1)).cuda()
    out = torch.full_like(tq, 77.0)
    s.batch.reserve(s.cache, nh)
    kv4.kvAttn(out, tq, s.cache, s.batch, nh, causal=causal, scale=1e36)
    torch.cuda.synchronize()
    check(out.cpu().numpy().reshape(s.m, nh, d).astype(np.float64), want, tol, "f32")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,group,d,page,lens,rows,causal", PATHS)
def test_the_largest_scales(kv4, heads, group, d, page, lens, rows, causal, dtype):
    """A scale near the end of f32 with small q and K: the largest score decides."""
    say(f"largest scales {heads}x{group}x{d} {lens} {dtype}")
    rng = np.random.default_rng(sum(lens) + 6)
    s = Setup(kv4, rng, heads, d, page, lens, rows)
    s.fill(rng, spread=1e-5)
    nh, scale = heads * group, float(np.float32(3e38))
    q = (rng.uniform(-1, 1, (s.m, nh, d)) * 2.0 ** -10).astype(NP[dtype])
    alone = rows_of_one_key(s, q, nh, causal, scale)
    assert alone.mean() > 0.5
    want, tol = one_key_outputs(s, q, nh, causal, dtype, scale)
    tq = torch.from_numpy(q.reshape(s.m, -1)).cuda()
    out = torch.full_like(tq, 77.0)
    s.batch.reserve(s.cache, nh)
    kv4.kvAttn(out, tq, s.cache, s.batch, nh, causal=causal, scale=scale)
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(s.m, nh, d).astype(np.float64)
    assert np.all(np.isfinite(got))
    check(got[alone], want[alone], tol[alone], dtype)


@pytest.mark.parametrize("score", [2.0 ** 20 - 20, 2.0 ** 20 - 10, 2.0 ** 20 - 3, 2.0 ** 20 + 4, -(2.0 ** 20) - 3, 2.0 ** 24,
                                   2.0 ** 27 + 2.0 ** 20, -(2.0 ** 28)])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,group,d,page,lens,rows,causal", PATHS[1:4])
def test_small_values_under_large_scores(kv4, heads, group, d, page, lens, rows, causal, dtype, score):
    """Keys that are alike with scores (as powers of 2) around 2^20 and past it, V of 10^-5
    and 10^-6: its mean, to as many bits as elsewhere (test_gpu_kv4_values.py's bound)."""
    say(f"small V, scores {score:g} {heads}x{group}x{d} {lens} {dtype}")
    rng = np.random.default_rng(sum(lens) + 7)
    s = Setup(kv4, rng, heads, d, page, lens, rows)
    s.fill(rng)
    code = rng.integers(1, 8, d)
    for i, n in enumerate(lens):
        kq, ks, vq, vs, there = s.held[i]
        kq[:], ks[:] = code, 3.0
        v = rng.uniform(0.2, 1, (n, heads, d)) * (1e-5 if i % 2 else 2e-6)
        vq[:], vs[:] = R.quantise(v.astype(np.float32))
        for t in range(n):
            p, o = s.place(i, t)
            for h in range(heads):
                R.put(s.data, page, d, p, h, o, kq[t, h], ks[t, h], vq[t, h], vs[t, h])
    s.dev.copy_(torch.from_numpy(s.data))
    nh = heads * group
    scale = 2.0 ** -8
    while dtype == "f16" and abs(score) / (3.0 * code.sum() * scale * 1.4426950408889634) > 3e4:
        scale *= 4
    q = np.full((s.m, nh, d), score / (3.0 * code.sum() * scale * 1.4426950408889634)).astype(NP[dtype])
    tq = torch.from_numpy(q.reshape(s.m, -1)).cuda()
    s.batch.reserve(s.cache, nh)
    out = torch.full_like(tq, 77.0)
    kv4.kvAttn(out, tq, s.cache, s.batch, nh, causal=causal, scale=scale)
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(s.m, nh, d).astype(np.float64)
    for i, n in enumerate(lens):
        v = R.value(s.held[i][2], s.held[i][3])
        for r, pos in enumerate(R.rows_of(n, rows[i])):
            k = pos + 1 if causal else n
            if k <= 0:
                continue
            o, a = (x.repeat(group, 0) for x in (v[:k].mean(0), np.abs(v[:k]).mean(0)))
            tol = ((2.0 ** -10 if dtype == "f16" else 3 * 2.0 ** -22) + 32 * 2.0 ** -23 + (n / 32 + 64) * 2.0 ** -24) * a
            tol += 2.0 ** -11 * np.abs(o) + 2.0 ** -25 if dtype == "f16" else 2.0 ** -24 * np.abs(o)
            tol += 7 * float(s.held[i][3].astype(np.float64).max()) * n * 2.0 ** -31
            worst = (np.abs(got[s.off[i] + r] - o) / tol).max()
            assert worst <= 1, (i, r, worst)
