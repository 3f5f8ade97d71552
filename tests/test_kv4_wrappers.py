"""What the 4-bit cache's wrappers hold on to and refuse, without a GPU."""
import weakref

import pytest

import kv4_ref as R
import madi_amd
from madi_amd import kv4

torch = pytest.importorskip("torch")


def pool(heads=2, dim=64, page=16, n_pages=4):
    return kv4.KV4(torch.zeros(n_pages * heads * R.block_bytes(page, dim), dtype=torch.uint8), page, heads, dim)


def indices(b=1, max_pages=8192):
    return torch.zeros(b, max_pages, dtype=torch.int32), torch.zeros(b, dtype=torch.int32)


def test_a_larger_workspace_leaves_the_smaller_one_where_it_is():
    """A captured graph, or a call still running on another stream, points to the
    workspace that a batch had then: it lives as long as the batch."""
    batch = kv4.Batch(*indices(), rows=1)
    small = batch.reserve(pool(), nh=2)
    assert small == batch._c.work_bytes > 0
    first, at = weakref.ref(batch.work), batch._c.work
    large = batch.reserve(pool(dim=256), nh=2)
    assert large == batch._c.work_bytes > small and batch._c.work == batch.work.data_ptr() != at
    assert first() is not None and first().data_ptr() == at
    now = batch.work
    assert batch.reserve(pool(), nh=2) == small and batch.work is now and batch._c.work_bytes == large


class Library:
    """The library as it is once madi_init has found a device, calls without effect."""

    def __init__(self):
        self.made = []

    def madi_device_cu_count(self):
        return 256

    def __getattr__(self, name):
        return lambda *args: self.made.append(name)


def test_tensors_in_host_memory_are_refused_once_there_is_a_device(monkeypatch):
    """A kernel that reads a host address faults the device: no such call is made."""
    cache, batch = pool(), kv4.Batch(*indices(2, 2), rows=3)
    k = torch.zeros(6, 128)
    calls = (lambda c, b: kv4.kvStore(c, b, k, k.clone()), lambda c, b: kv4.kvLoad(c, b, k, k.clone()),
             lambda c, b: kv4.kvAttn(k, k.clone(), c, b, nh=2))
    device = Library()
    real = kv4.lib()
    monkeypatch.setattr(kv4, "calls", device)
    for f in calls:
        f(cache, batch)
    assert device.made == ["madi_kv4_store", "madi_kv4_load", "madi_kv4_attn"]  # (which say that there is no device)
    monkeypatch.setattr(kv4, "lib", lambda: device)
    device.made.clear()
    for f in calls:
        with pytest.raises(madi_amd.MadiError) as e:
            f(cache, batch)
        assert e.value.code == -9 and "memory" in str(e.value)
    # tensors on the device, those of the call's rows not
    here = kv4.KV4.__new__(kv4.KV4)
    here.__dict__.update(cache.__dict__, on=0)
    there = kv4.Batch.__new__(kv4.Batch)
    there.__dict__.update(batch.__dict__, on=0)
    for f in calls:
        for c, b in ((here, batch), (cache, there), (here, there)):
            with pytest.raises(madi_amd.MadiError):
                f(c, b)
    assert not device.made and real is not device


def test_indices_on_two_devices_are_refused():
    table, lens = indices(2, 2)
    for args in ((table, lens.to("meta")), (table.to("meta"), lens)):
        with pytest.raises(madi_amd.MadiError) as e:
            kv4.Batch(*args)
        assert e.value.code == -9
    with pytest.raises(madi_amd.MadiError):
        kv4.Batch(table, lens, row_off=torch.zeros(3, dtype=torch.int32, device="meta"), m=2)


def test_reserve_refuses_head_counts_that_attention_refuses():
    batch = kv4.Batch(*indices(), rows=1)
    for nh in (0, 3, -2, 1, (1 << 32) + 2):
        with pytest.raises(madi_amd.MadiError) as e:
            batch.reserve(pool(), nh=nh)
        assert e.value.code == -5
    assert batch.work is None and batch.reserve(pool(), nh=6) > 0
