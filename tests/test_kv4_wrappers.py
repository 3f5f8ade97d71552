"""What the 4-bit cache's wrappers hold on to and refuse, without a GPU."""
import weakref

import pytest

import kv4_ref as R
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
