"""A Search or Adapters in other memory than the library's GPU's (made in host memory or before the library had
found its GPU), called with tensors that are where they should be: refused, without a GPU."""
import pytest

import madi_amd
from madi_amd import beam, kv4, lora

torch = pytest.importorskip("torch")


class Library:
    """The library once it has found a device: nothing is called."""

    def madi_device_cu_count(self):
        return 256

    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


def half(*shape):
    return torch.zeros(*shape, dtype=torch.float16)


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_objects_in_host_memory(monkeypatch):
    s = beam.Search(2, 3, 100, device="cpu")
    ad = lora.Adapters(half(2, 8, 64), half(2, 32, 8), torch.zeros(2))
    ad.reserve(5)
    w = madi_amd.q8.Q8(0, 0)
    library = Library()
    for module in (kv4, beam, lora):
        monkeypatch.setattr(module, "lib", lambda: library)
        monkeypatch.setattr(module, "calls", library)
    for module in (kv4, beam):
        monkeypatch.setattr(module, "DEVICE", -1)  # every tensor of a call counts as the GPU's
    for f in (lambda: beam.beamSelect(s, torch.zeros(6, 100), torch.zeros(2, 3)),
              lambda: lora.pprojLora(torch.zeros(5, 64), w, torch.zeros(5, 32), 5, 32, 64, ad, ints(5)),
              lambda: lora.pprojLora(torch.zeros(5, 64), w, torch.zeros(5, 32), 5, 32, 64, ad, ints(3), ints(5))):
        with pytest.raises(madi_amd.MadiError, match="ARG"):
            f()
