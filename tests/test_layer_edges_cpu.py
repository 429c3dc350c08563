"""CPU tests of what the operators beside the delta rule refuse or look at before any device work."""

from __future__ import annotations

import contextlib
import ctypes
import types

import pytest
import torch
from torch.autograd import forward_ad

from prometheus_amd import _native, kernels, serving


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


@pytest.mark.parametrize("who", [0, 1, 2])
def test_steps_do_not_drop_gradients(who):
    """A single token is forward only: while autograd records it is refused, not returned without a
    graph. The states stay as they were."""
    args = [torch.ones(2, 4), torch.zeros(2, 4), torch.ones(2, 4)]
    args[who].requires_grad_(True)
    with pytest.raises(kernels.KernelError, match="forward only"):
        kernels.linear_recurrence_step(*args)
    assert torch.equal(args[2], torch.ones(2, 4))
    if who < 2:
        cache = serving.RecurrenceStateCache(1, 2, 4, device="cpu")
        with pytest.raises(ValueError, match="forward only"):
            cache.decode(0, torch.zeros(2, dtype=torch.int32), *args[:2])
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):  # (the next check)
            cache.decode(0, torch.zeros(2, dtype=torch.int32), *args[:2])


def test_a_table_s_gradient_is_not_dropped():
    q = torch.ones(1, 3, 2, 4)
    table = kernels.rotation_table(3, 4, device="cpu").requires_grad_(True)
    with pytest.raises(kernels.KernelError, match="table"):
        kernels.norm_rotate(q, q, table)


def test_a_table_without_rows_is_no_null_pointer():
    L, p = _native.lib(), ctypes.c_void_p(16)  # (never dereferenced: there are no tokens)
    strides = (ctypes.c_int64 * 6)(0, 256, 64, 0, 256, 64)
    for rows, want in ((0, 0), (1, _native.E_NULL)):
        shared = (2, 0, 4, 4, 64, 64, rows, strides, 0, 0, 0, 1e-6, 0, 0, 0)
        assert L.pm_norm_rotate(p, p, None, None, None, None, p, p, *shared, None) == want
        assert L.pm_norm_rotate_bwd(p, p, None, None, None, None, p, p, p, p, None, None, *shared, None, 0, None) == want


def test_tangents_are_refused():
    """A dual tensor's tangent is not passed by, with and without reverse mode beside it."""
    x, q, s = torch.zeros(1, 3, 4), torch.ones(1, 3, 2, 4), torch.zeros(1, 4)
    cache = serving.RecurrenceStateCache(1, 1, 4, device="cpu")
    beta, one = torch.ones(1, 3, 2), torch.zeros(1, dtype=torch.int32)
    with forward_ad.dual_level():
        dual, heads = forward_ad.make_dual(x, x), forward_ad.make_dual(q, q)
        calls = [
            lambda: kernels.linear_recurrence(dual, x),
            lambda: kernels.linear_recurrence(x, dual),
            lambda: kernels.linear_recurrence(x, x, forward_ad.make_dual(s, s)),
            lambda: kernels.linear_recurrence_varlen(dual, x, [0, 3]),
            lambda: kernels.linear_recurrence_step(dual[:, 0], x[:, 0], s),
            lambda: cache.prefill(0, [0], dual, x),
            lambda: cache.decode(0, one, dual[:, 0], x[:, 0]),
            lambda: kernels.norm_rotate(q, heads),
            lambda: kernels.norm_rotate(q, q, q_weight=heads[0, 0, 0]),
            lambda: kernels.chunked_delta_rule(q, heads, q, beta),
        ]
        for i, call in enumerate(calls):
            with pytest.raises(kernels.KernelError, match="forward-mode"):
                call()
                pytest.fail(f"call {i} was not refused")
            with torch.no_grad(), pytest.raises(kernels.KernelError, match="forward-mode"):
                call()


def test_decode_runs_on_the_pool_s_device(monkeypatch):
    """Both caches launch with the pool's device as the current one, whichever is current outside."""
    inside = []

    @contextlib.contextmanager
    def on(device):
        inside.append(device)
        yield
        inside.pop()

    launched = []

    class Library:
        def __getattr__(self, name):
            return lambda *args: launched.append((name, list(inside))) or 0

    monkeypatch.setattr(kernels, "_on", on)
    monkeypatch.setattr(kernels, "_stream", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=0))
    monkeypatch.setattr(_native, "lib", Library)
    slots = torch.zeros(2, dtype=torch.int32)
    vectors = serving.RecurrenceStateCache(1, 2, 4, device="cpu")
    matrices = serving.LinearStateCache(1, 2, 3, 4, device="cpu")
    for cache in (vectors, matrices):
        monkeypatch.setattr(cache, "_check_cuda", lambda *tensors: None)
    vectors.decode(0, slots, torch.zeros(2, 4), torch.zeros(2, 4))
    x = torch.zeros(2, 3, 4)
    matrices.decode(0, slots, x, x, x, torch.zeros(2, 3))
    cpu = torch.device("cpu")
    assert launched == [("pm_linear_recurrence_step", [cpu]), ("pm_delta_step_slots", [cpu])]


def test_a_weight_that_is_not_there_has_no_gradient():
    """The C entry used to write zeros where a NULL weight's gradient was asked for."""
    L, p = _native.lib(), ctypes.c_void_p(16)  # never dereferenced: validation fails first
    strides = (ctypes.c_int64 * 6)(120, 24, 6, 30, 6, 6)
    need = L.pm_norm_rotate_bwd_workspace_bytes(2, 5, 4, 1, 6)
    for wq, wk, gwq, gwk in ((None, p, p, None), (p, None, None, p), (None, None, p, p)):
        rc = L.pm_norm_rotate_bwd(p, p, None, None, wq, wk, p, p, p, p, gwq, gwk, 2, 5, 4, 1, 6, 0, 0, strides, 0, 0, 0,
                                  1e-6, 0, 0, 0, p, need, None)
        assert rc == _native.E_NULL and b"weight" in L.pm_last_error()
