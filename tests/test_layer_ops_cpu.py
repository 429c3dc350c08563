"""CPU tests of the operators beside the delta rule: what they refuse before any device work, and
the 64-bit forms that the GPU tests compare with (against each other and against differences)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import layer_oracle as ref
from prometheus_amd import _native, kernels, serving

P = ctypes.c_void_p(16)  # never dereferenced: validation fails first


# --- the 64-bit forms ---


@pytest.mark.parametrize("T,state", [(1, True), (7, False), (40, True)])
def test_recurrence_gradients_against_differences(T, state):
    rng = np.random.default_rng(T)
    x, g = rng.normal(size=(2, T, 3)), -rng.random((2, T, 3))
    s0 = rng.normal(size=(2, 3)) if state else None
    gh, gs = rng.normal(size=x.shape), rng.normal(size=(2, 3))

    def loss(x, g, s0):
        h, s = ref.recurrence(x, g, s0)
        return np.sum(gh * h) + np.sum(gs * s)

    gx, gg, gs0 = ref.recurrence_bwd(x, g, s0, gh, gs)
    e = 1e-6
    for got, at in ((gx, 0), (gg, 1), (gs0, 2)):
        args = [x, g, s0]
        if args[at] is None:
            continue
        v = rng.normal(size=args[at].shape)
        up, down = list(args), list(args)
        up[at], down[at] = args[at] + e * v, args[at] - e * v
        diff = (loss(*up) - loss(*down)) / (2 * e)
        assert diff == pytest.approx(np.sum(got * v), rel=1e-6, abs=1e-6)


@pytest.mark.parametrize("norm", ["l2", "rms"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("R", [0, 4, 6])
def test_head_norm_gradients_against_differences(norm, interleaved, R):
    rng = np.random.default_rng(R)
    x, gz, w = rng.normal(size=(5, 2, 6)), rng.normal(size=(5, 2, 6)), 1 + 0.1 * rng.normal(size=6)
    table = rng.normal(size=(9, R)) if R else None
    pos = rng.integers(0, 9, 5)

    def loss(x, w):
        return np.sum(gz * ref.head_norm(x, table, pos, norm, w, 1e-6, interleaved))

    gx, gw = ref.head_norm_bwd(x, gz, table, pos, norm, w, 1e-6, interleaved)
    e, v, vw = 1e-6, rng.normal(size=x.shape), rng.normal(size=6)
    assert (loss(x + e * v, w) - loss(x - e * v, w)) / (2 * e) == pytest.approx(np.sum(gx * v), rel=1e-6)
    assert (loss(x, w + e * vw) - loss(x, w - e * vw)) / (2 * e) == pytest.approx(np.sum(gw * vw), rel=1e-6)


def test_rotation_table_is_exact_far_out():
    t = kernels.rotation_table(40000, 64, device="cpu").numpy()
    i = np.arange(32)
    angle = 39999.0 * 10000.0 ** (-2.0 * i / 64)
    np.testing.assert_allclose(t[-1], np.concatenate([np.cos(angle), np.sin(angle)]), atol=2e-7)
    for bad in ((3, 5), (3, 0), (-1, 4)):
        with pytest.raises(kernels.KernelError):
            kernels.rotation_table(*bad, device="cpu")


# --- refusals before any device work ---


def test_recurrence_shape_checks():
    x = np.zeros((2, 5, 3), np.float32)
    bad = [
        lambda: kernels.linear_recurrence(x, x[:, :4]),
        lambda: kernels.linear_recurrence(x[0], x[0]),
        lambda: kernels.linear_recurrence(x, x, np.zeros((2, 4), np.float32)),
        lambda: kernels.linear_recurrence(x, x, out_dtype="fp16"),
        lambda: kernels.linear_recurrence_fwd(x, x[:1]),
        lambda: kernels.linear_recurrence_varlen(x, x, [0, 5]),  # a batch of two is not packed
        lambda: kernels.linear_recurrence_varlen(x[0], x[0], [0, 4]),
        lambda: kernels.linear_recurrence_varlen(x[0], x[0], [1, 5]),
        lambda: kernels.linear_recurrence_varlen(x[0], x[0], [0, 4, 3, 5]),
        lambda: kernels.linear_recurrence_varlen(x[0], x[0], [0.0, 5.0]),
        lambda: kernels.linear_recurrence_varlen(x[0], x[0], [0, 5], np.zeros((2, 3), np.float32)),
        lambda: kernels.linear_recurrence_varlen(torch.zeros(5, 3, requires_grad=True), torch.zeros(5, 3), [0, 5]),
        lambda: kernels.linear_recurrence_step(x[:, 0], x[:, 0], None),
        lambda: kernels.linear_recurrence_step(x[:, 0], x[:, 0], np.zeros((2, 4), np.float32)),
        lambda: kernels.linear_recurrence_step(x[:, 0], x[:, 0], np.zeros((2, 3))),
        lambda: kernels.linear_recurrence_step(x, x, np.zeros((2, 3), np.float32)),
    ]
    res = kernels.recurrence._RecurrenceResidual(x, x, np.zeros((2, 1, 3), np.float32), torch.float32)
    bad += [
        lambda: kernels.linear_recurrence_bwd(res, (x[:, :4], None)),
        lambda: kernels.linear_recurrence_bwd(res, (None, x[:, 0, :2])),
        lambda: kernels.linear_recurrence_bwd(
            kernels.recurrence._RecurrenceResidual(x, x, np.zeros((2, 2, 3), np.float32), torch.float32), (x, None)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(kernels.KernelError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_head_norm_shape_checks():
    q, k = np.zeros((2, 5, 4, 6), np.float32), np.zeros((2, 5, 1, 6), np.float32)
    t = np.zeros((5, 4), np.float32)
    f = kernels.norm_rotate
    bad = [
        lambda: f(q, k[:, :4]),
        lambda: f(q, k[..., :5]),
        lambda: f(q[0, 0], k[0, 0]),
        lambda: f(q, k, norm="max"),
        lambda: f(q, k, eps=-1.0),
        lambda: f(q, k, eps=float("nan")),
        lambda: f(q, k, q_weight=np.ones(5, np.float32)),
        lambda: f(q, k, k_weight=np.ones((1, 6), np.float32)),
        lambda: f(q, k, np.zeros((5, 3), np.float32)),  # odd
        lambda: f(q, k, np.zeros((5, 8), np.float32)),  # wider than the head
        lambda: f(q, k, np.zeros(4, np.float32)),
        lambda: f(q, k, t[:4]),  # five tokens, four rows
        lambda: f(q, k, None, np.zeros(5, np.int64)),  # positions without a table
        lambda: f(q, k, t, np.zeros(4, np.int64)),
        lambda: f(q, k, t, np.zeros((1, 5), np.int64)),
        lambda: f(q, k, t, np.zeros(5)),
        lambda: f(q, k, t, [0, 1, 2, 3, 5]),
        lambda: f(q, k, t, torch.tensor([0, 1, 2, 3, -1])),
        lambda: f(q[0], k[0], t),  # packed tokens need positions
        lambda: f(np.zeros((1, 1, 1, 257), np.float32), np.zeros((1, 1, 1, 257), np.float32)),
        lambda: f(np.zeros((1, 1, 1, 0), np.float32), np.zeros((1, 1, 1, 0), np.float32)),
    ]
    res = kernels.head_norm._NormRotateResidual(q, k, None, None, None, None, "l2", 1e-6, False)
    bad.append(lambda: kernels.norm_rotate_bwd(res, (k, None)))
    for i, call in enumerate(bad):
        with pytest.raises(kernels.KernelError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_recurrence_abi_argument_validation_without_gpu():
    L = _native.lib()

    def fwd(x=P, g=P, cu=None, s0=None, slots=None, n_slots=0, bad=None, h=P, s=P, kept=None, n=2, T=5, C=3,
            st=(15, 3, 15, 3), types=(0, 0, 0)):
        return L.pm_linear_recurrence(x, g, cu, s0, slots, n_slots, bad, h, s, kept, n, T, C, *st, *types, None, 0, None)

    assert fwd(types=(0, 1, 0)) == fwd(types=(2, 0, 0)) == fwd(types=(0, 0, 5)) == _native.E_DTYPE
    assert fwd(n=-1) == fwd(T=-1) == fwd(C=-1) == fwd(st=(-1, 3, 15, 3)) == fwd(st=(15, 3, 15, 1 << 50)) == _native.E_SHAPE
    assert fwd(n=2**31 - 1, T=2**31 - 1, C=2**31 - 1) == fwd(cu=P, n=2**31 - 1, C=2**31 - 1, T=0) == _native.E_SHAPE
    assert fwd(x=None) == fwd(g=None) == fwd(h=None) == fwd(s=None) == _native.E_NULL
    assert fwd(x=ctypes.c_void_p(18)) == fwd(cu=ctypes.c_void_p(18)) == fwd(s0=ctypes.c_void_p(18)) == _native.E_ALIGN
    assert fwd(types=(1, 1, 1), h=ctypes.c_void_p(17)) == _native.E_ALIGN
    assert fwd(slots=P, n_slots=4) == fwd(slots=P, n_slots=-1, s0=P) == _native.E_SHAPE  # s0 is not s_out
    assert fwd(cu=P, kept=P) == _native.E_UNSUPPORTED
    assert b"kept" in L.pm_last_error()
    assert fwd(n=0) == fwd(C=0) == 0  # nothing to do, nothing touched

    def bwd(x=P, kept=P, gh=P, gs=None, gx=P, gg=P, gs0=P, B=2, T=5, C=3, st=(15, 3, 15, 3), types=(0, 0, 0)):
        return L.pm_linear_recurrence_bwd(x, P, kept, gh, gs, gx, gg, gs0, B, T, C, *st, *types, None, 0, None)

    assert bwd(types=(0, 1, 0)) == _native.E_DTYPE
    assert bwd(B=-1) == bwd(st=(15, -3, 15, 3)) == _native.E_SHAPE
    assert bwd(x=None) == bwd(kept=None) == bwd(gx=None) == bwd(gg=None) == bwd(gs0=None) == _native.E_NULL
    assert bwd(gs=ctypes.c_void_p(18)) == bwd(gh=ctypes.c_void_p(18)) == _native.E_ALIGN
    assert bwd(B=0) == bwd(C=0) == 0

    def step(s=P, slots=None, n_slots=0, x=P, h=P, B=2, C=3, st=(3, 3), types=(0, 0, 0)):
        return L.pm_linear_recurrence_step(s, slots, n_slots, x, P, h, B, C, *st, *types, None)

    assert step(types=(0, 0, 3)) == _native.E_DTYPE
    assert step(B=-1) == step(st=(-1, 3)) == step(slots=P, n_slots=-1) == _native.E_SHAPE
    assert step(s=None) == step(x=None) == step(h=None) == _native.E_NULL
    assert step(s=ctypes.c_void_p(18)) == _native.E_ALIGN
    assert step(B=0) == step(C=0) == 0


def test_head_norm_abi_argument_validation_without_gpu():
    L = _native.lib()
    strides = (ctypes.c_int64 * 6)(120, 24, 6, 30, 6, 6)

    def args(q=P, table=None, pos=None, wq=None, sizes=(2, 5, 4, 1, 6, 0, 0), strides=strides, sb=0, pos64=0, norm=0,
             eps=1e-6, dtype=0, w=0):
        return (q, P, table, pos, wq, None), (*sizes, strides, sb, pos64, norm, eps, 0, dtype, w)

    def fwd(out=P, **kw):
        a, b = args(**kw)
        return L.pm_norm_rotate(*a, out, P, *b, None)

    assert fwd(dtype=2) == fwd(w=7) == _native.E_DTYPE
    for sizes in ((-1, 5, 4, 1, 6, 0, 0), (2, 5, 4, 1, 0, 0, 0), (2, 5, 4, 1, 257, 0, 0), (2, 5, 4, 1, 6, 3, 9),
                  (2, 5, 4, 1, 6, 8, 9), (2, 5, 4, 1, 6, -2, 9), (2**31 - 1, 2**31 - 1, 4, 1, 6, 0, 0),
                  (1, 1, 2**31 - 1, 1, 6, 0, 0)):
        assert fwd(sizes=sizes) == _native.E_SHAPE, sizes
    assert fwd(sizes=(2, 5, 4, 1, 6, 4, -1), table=P) == _native.E_SHAPE
    assert fwd(norm=2) == fwd(eps=-1.0) == fwd(eps=float("nan")) == fwd(sb=-1) == _native.E_SHAPE
    assert fwd(strides=(ctypes.c_int64 * 6)(120, 24, 6, 30, -6, 6)) == _native.E_SHAPE
    assert fwd(q=None) == fwd(out=None) == fwd(strides=None) == fwd(sizes=(2, 5, 4, 1, 6, 4, 9)) == _native.E_NULL
    odd = ctypes.c_void_p(18)
    assert fwd(q=odd) == fwd(wq=odd) == fwd(out=odd) == fwd(table=odd, sizes=(2, 5, 4, 1, 6, 4, 9)) == _native.E_ALIGN
    assert fwd(table=P, pos=ctypes.c_void_p(20), pos64=1, sizes=(2, 5, 4, 1, 6, 4, 9)) == _native.E_ALIGN
    assert fwd(sizes=(0, 5, 4, 1, 6, 0, 0)) == fwd(sizes=(2, 0, 4, 1, 6, 0, 0)) == 0

    def bwd(gq=P, gw=None, ws=None, n=0, **kw):
        a, b = args(**kw)
        return L.pm_norm_rotate_bwd(*a, P, P, gq, P, gw, None, *b, ws, n, None)

    need = L.pm_norm_rotate_bwd_workspace_bytes(2, 5, 4, 1, 6)
    assert need > 0 and L.pm_norm_rotate_bwd_workspace_bytes(-1, 5, 4, 1, 6) == 0
    assert bwd(gq=None) == _native.E_NULL
    assert bwd(gw=odd) == bwd(gq=odd) == _native.E_ALIGN
    assert bwd(gw=P) == bwd(gw=P, ws=P, n=need - 1) == bwd(gw=P, ws=ctypes.c_void_p(20), n=need) == _native.E_WORKSPACE
    assert bwd(sizes=(0, 5, 4, 1, 6, 0, 0)) == 0


def test_recurrence_cache_bookkeeping_without_gpu():
    cache = serving.RecurrenceStateCache(2, 3, 4, device="cpu")
    assert cache.pool.shape == (2, 3, 4) and cache.alloc(2) == [0, 1] and cache.n_free == 1
    cache._pool[:] = 1.0
    cache.free([0])
    assert cache.alloc(1) == [0] and not cache.pool[:, 0].any() and cache.pool[:, 1].all()
    x = torch.zeros(2, 5, 4)
    for bad in (lambda: cache.prefill(2, [0, 1], x, x), lambda: cache.prefill(0, [0, 3], x, x),
                lambda: cache.prefill(0, [0, 0], x, x), lambda: cache.prefill(0, [0], x, x),
                lambda: cache.prefill(0, [0, 1], x[..., :3], x[..., :3])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        cache.prefill(0, [0, 1], x, x)
    with pytest.raises(RuntimeError):
        cache.decode(0, torch.zeros(2, dtype=torch.int32), x[:, 0], x[:, 0])
    with pytest.raises(ValueError):
        serving.RecurrenceStateCache(1, 1, 0, device="cpu")


def test_no_cpu_fallback():
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    x = np.zeros((1, 2, 3), np.float32)
    with pytest.raises(RuntimeError):
        kernels.linear_recurrence(x, x)
    with pytest.raises(RuntimeError):
        kernels.norm_rotate(x, x)
