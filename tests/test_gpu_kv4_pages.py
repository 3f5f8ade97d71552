"""The 4-bit cache with the largest pages: 2^20 tokens, of which only the last ones were
ever stored, read through a window; sequences that end in a page and just past it."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import NP, check, kv4, say  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

PAGE, KEPT, WINDOW = 1 << 20, 300, 100


@pytest.mark.parametrize("heads,group,d,rows", [(2, 4, 256, 3), (1, 2, 64, 1), (2, 32, 128, 190), (1, 5, 96, 37)])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_pages_of_2_to_20(kv4, heads, group, d, rows, dtype):
    say(f"large pages {heads}x{group}x{d} rows {rows} {dtype}")
    rng = np.random.default_rng(d + rows)
    lens = [PAGE - 3, PAGE + 50, 2 * PAGE]
    cache = kv4.alloc(5, PAGE, heads, d)
    cache.data.fill_(0xff)  # scales that are no numbers wherever nothing is stored
    table = torch.tensor([[4, 99], [0, 2], [1, 3]], dtype=torch.int32).cuda()
    dev_lens = torch.tensor(lens, dtype=torch.int32).cuda()
    x = rng.standard_normal((3 * KEPT, 2, heads, d), dtype=np.float32).astype(np.float16)
    kv = torch.from_numpy(x).cuda()
    kv4.kvStore(cache, kv4.Batch(table, dev_lens, rows=KEPT), kv[:, 0], kv[:, 1])
    k, v = torch.empty(2, 3 * KEPT, heads * d, dtype=torch.float16, device="cuda")
    kv4.kvLoad(cache, kv4.Batch(table, dev_lens, rows=KEPT), k, v)
    torch.cuda.synchronize()
    for j, got in enumerate((k, v)):
        want = R.value(*R.quantise(x[:, j]))
        assert np.array_equal(got.cpu().numpy().reshape(want.shape), want.astype(np.float16))
    nh = heads * group
    q = rng.standard_normal((3 * rows, nh, d), dtype=np.float32).astype(NP[dtype])
    want, tol = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(3):
        own = x[i * KEPT:(i + 1) * KEPT]
        for h in range(heads):
            kq, ks, vq, vs = *R.quantise(own[:, 0, h]), *R.quantise(own[:, 1, h])
            r, c = slice(i * rows, (i + 1) * rows), slice(h * group, (h + 1) * group)
            o, a, v1 = R.attention(q[r, c], R.value(kq, ks), R.value(vq, vs), np.ones(KEPT, bool),
                                   list(range(KEPT - rows, KEPT)), True, WINDOW, d ** -0.5)
            e = R.score_error(q[r, c], ks, d ** -0.5)[..., None]
            n = 2 * (WINDOW + rows)
            unit, last = (2.0 ** -10, 2.0 ** -11 * np.abs(o) + 2.0 ** -25) if dtype == "f16" else \
                (3 * 2.0 ** -22, 2.0 ** -24 * np.abs(o))
            want[r, c] = o
            tol[r, c] = (unit + 2 * e + 32 * 2.0 ** -23 + (n / 32 + 64) * 2.0 ** -24) * a + last + 2.0 ** -32 * v1
    tq = torch.from_numpy(q.reshape(3 * rows, -1)).cuda()
    batch = kv4.Batch(table, dev_lens, rows=rows)
    batch.reserve(cache, nh)
    out = torch.full_like(tq, 77.0)
    kv4.kvAttn(out, tq, cache, batch, nh, window=WINDOW)
    torch.cuda.synchronize()
    check(out.cpu().numpy().reshape(q.shape).astype(np.float64), want, tol, dtype)
