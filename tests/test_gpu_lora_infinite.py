"""Projections with adapters whose A x holds infinities, in 64 bits and on the GPU: the same infinities, the same NaN
(an infinity against a zero of B), the rest as close as without them."""
import numpy as np
import pytest

import serving_ref as S
from test_gpu_lora import Case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def q8():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import madi_amd.q8 as q8
    q8.init()
    return q8


@pytest.mark.parametrize("m,n,k,rank", [(7, 320, 256, 8), (24, 320, 640, 16), (40, 1280, 5120, 24), (200, 160, 192, 40),
                                        (300, 1280, 1280, 64), (700, 2048, 320, 16), (700, 640, 2112, 128)])
def test_infinite_products(q8, m, n, k, rank):
    """One rank of one adapter is infinite in its rows, of either sign, beside numbers past f16's range."""
    c = Case(q8, m, n, k, rank, 4, seed=m + n, big=1000.0)
    c.x = np.clip(c.x, -6e4, 6e4)
    c.x[:, 5] = np.where(np.arange(m) % 2, 2.0, -3.0)
    c.a[1] *= np.float16(50)
    c.a[1, rank - 3, 5] = np.inf
    c.a[2, 1] = 0
    c.a[2, 1, 5] = -np.inf          # (0 against the other rows' numbers)
    c.b[1, 7:11, rank - 3] = 0
    c.dx.copy_(torch.from_numpy(c.x))
    c.ad = c.lora.Adapters(torch.from_numpy(c.a).cuda(), torch.from_numpy(c.b).cuda(), c.ad.scale)
    a = np.arange(m) % 5 - 1
    with np.errstate(invalid="ignore"):
        ref, size = S.lora(c.x, c.q, c.s, c.a, c.b, c.scale, a)
    got = c.run(a).cpu().numpy().astype(np.float64)
    assert np.isinf(ref).any() and np.isnan(ref).any() and (ref == np.inf).any() and (ref == -np.inf).any()
    fine = np.isfinite(ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(got[np.isinf(ref)], ref[np.isinf(ref)])
    # every sum has at most k + rank additions of 2^-24, A x is kept to 22 bits
    err = np.abs(got[fine] - ref[fine])
    assert (err <= (k + rank + 8) * 2.0 ** -24 * size[fine]).all(), (err / size[fine]).max()
