"""What the 4-bit cache's wrappers refuse on a machine with a GPU: tensors in host
memory, before any of their addresses reaches a kernel."""
import pytest

import kv4_ref as R
import madi_amd
from test_gpu_kv4 import kv4, say  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_host_memory(kv4):
    say("host memory")
    data = torch.zeros(4 * 2 * R.block_bytes(16, 64), dtype=torch.uint8)
    table, lens = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32), torch.tensor([20, 9], dtype=torch.int32)
    row_off = torch.tensor([0, 2, 3], dtype=torch.int32)
    k = torch.zeros(3, 128)
    on = lambda *t: [x.cuda() for x in t]
    cache, host_cache = (kv4.KV4(d, page=16, heads=2, dim=64) for d in (data.cuda(), data))
    batch = kv4.Batch(*on(table, lens), rows=2, row_off=row_off.cuda(), m=3)
    host_batch = kv4.Batch(table, lens, rows=2, row_off=row_off, m=3)
    for args in ((table.cuda(), lens), (table, lens.cuda())):
        with pytest.raises(madi_amd.MadiError) as e:
            kv4.Batch(*args, rows=2)
        assert e.value.code == -9
    with pytest.raises(madi_amd.MadiError):
        kv4.Batch(*on(table, lens), rows=2, row_off=row_off, m=3)
    dk, dv = on(k, k)
    for c, b, x, y in ((host_cache, batch, dk, dv), (cache, host_batch, dk, dv), (host_cache, host_batch, k, k),
                       (cache, batch, k, dv), (cache, batch, dk, k)):
        for f in (lambda: kv4.kvStore(c, b, x, y), lambda: kv4.kvLoad(c, b, x, y),
                  lambda: kv4.kvAttn(x, y, c, b, nh=2)):
            with pytest.raises(madi_amd.MadiError) as e:
                f()
            assert e.value.code == -9
    kv4.kvStore(cache, batch, dk, dv)
    kv4.kvLoad(cache, batch, dk, dv)
    kv4.kvAttn(dk, dv, cache, batch, nh=2)
    torch.cuda.synchronize()
    assert torch.equal(dk, torch.zeros_like(dk))
