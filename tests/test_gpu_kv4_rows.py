"""What the 4-bit cache's calls leave beside the rows that they write: a deferred
dequantisation's result in the same memory, and other rows where one holds no numbers."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import NP, Setup, attend, check, kv4, say  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("call", ["store", "load", "attn"])
def test_a_deferred_weight_around_the_rows(kv4, call):
    """kDeq into a scratch, of which a store, load or attention then writes some rows and
    columns: the rest is the weight."""
    from madi_amd import q8
    say(f"deferred weight, {call}")
    rng = np.random.default_rng(41)
    n, k, heads, d, page = 256, 512, 2, 64, 16
    w = q8.upload_q8(rng.integers(-127, 128, (n, k)).astype(np.int8), rng.uniform(0.01, 0.1, (n, k // 32)).astype(np.float16))
    q8.set_deferred_dequant(True)
    plain, scratch = torch.zeros(2, k, n, dtype=torch.float16, device="cuda")
    q8.kDeq(plain, w, n, k)
    q8.materialize(plain)
    s = Setup(kv4, rng, heads, d, page, [40, 33], [6, 9])
    s.fill(rng)
    # 40 rows in the call, of which the sequences have 3 .. 17
    b = kv4.Batch(s.batch.table, s.batch.lens, rows=9, row_off=torch.tensor([3, 9, 18], dtype=torch.int32).cuda(), m=40)
    src = torch.from_numpy(rng.standard_normal((2, 40, heads * d)).astype(np.float16)).cuda()
    q8.kDeq(scratch, w, n, k)
    if call == "store":
        cache = kv4.KV4(scratch, page, heads, d, s.n_pages)
        kv4.kvStore(cache, b, src[0], src[1])
    elif call == "load":
        kv4.kvLoad(s.cache, b, scratch[:40, :128], scratch[k - 40:, 128:])
    else:
        kv4.kvAttn(scratch[:40, :128], src[0], s.cache, b, heads)
    q8.materialize(scratch)
    q8.sync()
    torch.cuda.synchronize()
    want = plain.clone()
    if call == "store":
        cache = kv4.KV4(want, page, heads, d, s.n_pages)
        kv4.kvStore(cache, b, src[0], src[1])
    elif call == "load":
        kv4.kvLoad(s.cache, b, want[:40, :128], want[k - 40:, 128:])
    else:
        kv4.kvAttn(want[:40, :128], src[0], s.cache, b, heads)
    torch.cuda.synchronize()
    for t in (plain, scratch, want):
        q8.forget(t)
    changed = (want.view(torch.int16) != plain.view(torch.int16)).sum().item()
    assert 0 < changed < want.numel() // 4
    assert torch.equal(scratch.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,group,d,page,lens,rows", [
    (2, 4, 64, 16, [200, 33], [3, 5]), (1, 5, 128, 64, [3000, 2300], [4, 2]), (4, 64, 64, 16, [230, 233], [230, 233])])
def test_rows_that_hold_no_numbers(kv4, heads, group, d, page, lens, rows, dtype):
    """A query that is infinite or no number makes its own row and head NaN, or leaves it
    finite; the others are what they are without it."""
    say(f"rows of NaN {heads}x{group}x{d} {lens} {dtype}")
    rng = np.random.default_rng(sum(lens) + 42)
    s = Setup(kv4, rng, heads, d, page, lens, rows)
    s.fill(rng)
    nh = heads * group
    q = rng.standard_normal((s.m, nh, d)).astype(NP[dtype])
    want, tol = s.expect(q, nh, True, 0, d ** -0.5, dtype)
    bad = rng.random((s.m, nh)) < 0.2
    bad[0, 0] = True
    q[bad, 7] = rng.choice(np.array([np.nan, np.inf, -np.inf], NP[dtype]), int(bad.sum()))
    got = attend(s, q, nh, dtype)
    check(got[~bad], want[~bad], tol[~bad], dtype)
