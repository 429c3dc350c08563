"""CPU tests of what the operators beside the delta rule refuse or look at before any device work."""

from __future__ import annotations

import pytest
import torch

from prometheus_amd import kernels, serving


def test_cache_prefill_looks_at_the_offsets_device(monkeypatch):
    """Offsets of another GPU than x's are refused where all of a call's tensors are compared."""
    seen = []

    class Compared(Exception):
        pass

    def compare(*tensors):
        seen.extend(tensors)
        raise Compared

    cache = serving.RecurrenceStateCache(1, 2, 4, device="cpu")
    monkeypatch.setattr(cache, "_check_cuda", lambda *tensors: None)
    monkeypatch.setattr(kernels, "_Call", compare)
    x, cu = torch.zeros(5, 4), torch.tensor([0, 2, 5])
    with pytest.raises(Compared):
        cache.prefill(0, [0, 1], x, x, cu)
    assert any(t is cu for t in seen)
