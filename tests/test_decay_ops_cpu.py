"""CPU tests of decay attention and the norms around it: what they refuse before any device work, and
the 64-bit forms that the GPU tests compare with (against each other and against differences)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import decay_oracle as ref
from prometheus_amd import _native, kernels, serving
from prometheus_amd.kernels import row_norms

P = ctypes.c_void_p(16)  # never dereferenced: validation fails first
F64 = torch.float64


def normal(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=F64)


# --- the 64-bit forms ---


@pytest.mark.parametrize("T,Hq,H,gate", [(1, 1, 1, "token"), (9, 4, 2, "token"), (20, 2, 2, "head")])
@pytest.mark.parametrize("s0", [True, False])
def test_decay_gradients_against_differences(T, Hq, H, gate, s0):
    q, k, v = normal(2, T, Hq, 5), normal(2, T, H, 5, seed=1), normal(2, T, H, 5, seed=2)
    g = -torch.rand(*((2, T, H) if gate == "token" else (H,)), dtype=F64, generator=torch.Generator().manual_seed(3))
    x = [q, k, v, g, normal(2, H, 5, 5, seed=4) if s0 else None]
    go, gs = normal(2, T, Hq, 5, seed=5), normal(2, H, 5, 5, seed=6)

    def loss(*x):
        o, s = ref.decay(*x, scale=0.7)
        return ((go * o).sum() + (gs * s).sum()).item()

    grads = ref.decay_bwd(*x, go, gs, 0.7)
    for i, (a, got) in enumerate(zip(x, grads)):
        if a is None:
            continue
        assert got.shape == a.shape
        d, e = normal(*a.shape, seed=7 + i), 1e-6
        up, down = list(x), list(x)
        up[i], down[i] = a + e * d, a - e * d
        assert (loss(*up) - loss(*down)) / (2 * e) == pytest.approx((got * d).sum().item(), rel=1e-6, abs=1e-7)


def test_decay_without_decays_is_a_running_sum():
    q, k, v = normal(1, 6, 1, 3), normal(1, 6, 1, 3, seed=1), normal(1, 6, 1, 3, seed=2)
    o, s = ref.decay(q, k, v, torch.zeros(1))
    want = (torch.tril(q[0, :, 0] @ k[0, :, 0].T)) @ v[0, :, 0]
    assert torch.allclose(o[0, :, 0], want) and torch.allclose(s[0, 0], k[0, :, 0].T @ v[0, :, 0])


@pytest.mark.parametrize("activation", ["silu", "sigmoid"])
@pytest.mark.parametrize("first", [True, False])
def test_gated_norm_sizes_bound_the_gradients(activation, first):
    x, z, w, gy = normal(4, 9), normal(4, 9, seed=1), normal(9, seed=2), normal(4, 9, seed=3)
    options = {"activation": activation, "gate_first": first}
    grads = ref.gradients(lambda *a: ref.gated(*a, **options), (x, z, w), (gy,))
    for g, size in zip(grads, ref.gated_bwd_size(x, z, w, gy, **options)):
        assert (g.abs() <= size * (1 + 1e-12)).all()
    d, e = normal(4, 9, seed=4), 1e-6
    up, down = (ref.gated(x + s * e * d, z, w, **options) for s in (1, -1))
    assert ((up - down) / (2 * e) * gy).sum().item() == pytest.approx((grads[0] * d).sum().item(), rel=1e-6)


def test_residual_norm_sizes_bound_the_gradients():
    x, r, gy, gh = (normal(4, 9, seed=i) for i in range(4))
    w, wp = normal(9, seed=4), normal(9, seed=5)
    for p in (wp, None):
        grads = ref.gradients(lambda *a: ref.residual(*a, scale=0.5), (x, r, w, p), (gy, gh))
        for g, size in zip(grads, ref.residual_bwd_size(x, r, w, p, gy, gh, 0.5)):
            assert g is None or (g.abs() <= size * (1 + 1e-12)).all()


# --- refusals before any device work ---


def test_decay_shape_checks():
    q = np.zeros((2, 5, 4, 8), np.float32)
    k, g = q[:, :, :2], np.zeros((2, 5, 2), np.float32)
    s = np.zeros((2, 2, 8, 8), np.float32)
    call = kernels.decay_attention
    bad = [
        lambda: call(q, k, k[:, :4], g),
        lambda: call(q[:, :4], k, k, g),
        lambda: call(q[..., :7], k, k, g),
        lambda: call(q[:, :, :3], k, k, g),
        lambda: call(q[:, :, :0], k, k, g),
        lambda: call(q[0], k[0], k[0], g[0]),
        lambda: call(q, k, k, g[:, :, :1]),
        lambda: call(q, k, k, np.zeros(4, np.float32)),
        lambda: call(q, k, k, g, s[:1]),
        lambda: call(q, k, k, g, s, scale=float("nan")),
        lambda: call(q, k, k, g, out_dtype="fp16"),
        lambda: call(np.zeros((1, 1, 1, 257)), np.zeros((1, 1, 1, 257)), np.zeros((1, 1, 1, 257)), np.zeros(1)),
        lambda: kernels.decay_attention_varlen(q, k, k, g, [0, 5]),
        lambda: kernels.decay_attention_varlen(q[:1], k[:1], k[:1], g[:1], [0, 4]),
        lambda: kernels.decay_attention_varlen(q[0], k[0], k[0], g[0], [1, 5]),
        lambda: kernels.decay_attention_varlen(q[0], k[0], k[0], g[0], [0, 4, 3, 5]),
        lambda: kernels.decay_attention_varlen(q[0], k[0], k[0], g[0], [0.0, 5.0]),
        lambda: kernels.decay_attention_varlen(q[0], k[0], k[0], g[0], [0, 5], s),
        lambda: kernels.decay_attention_step(q[:, 0], k[:, 0], k[:, 0], g[:, 0], None),
        lambda: kernels.decay_attention_step(q[:, 0], k[:, 0], k[:, 0], g[:, 0], s.astype(np.float64)),
        lambda: kernels.decay_attention_step(q[:, 0], k[:, 0], k[:, 0], g[:, 0], s.tolist()),
        lambda: kernels.decay_attention_step(q[:, 0], k[:, 0], k[:, 0], g[:, 0], s[:1]),
    ]
    for f in bad:
        with pytest.raises(kernels.KernelError):
            f()


def test_decay_forward_only_calls_refuse_gradients():
    q, g = torch.zeros(1, 3, 2, 8), torch.zeros(2, requires_grad=True)
    for f in (lambda: kernels.decay_attention_varlen(q, q, q, g, [0, 3]),
              lambda: kernels.decay_attention_step(q[:, 0], q[:, 0], q[:, 0], g, torch.zeros(1, 2, 8, 8))):
        with pytest.raises(kernels.KernelError, match="forward only"):
            f()


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd

    x = torch.zeros(1, 3, 2, 8)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for f in (lambda: kernels.decay_attention(dual, x, x, torch.zeros(2)), lambda: kernels.gated_norm(dual, x),
                  lambda: kernels.residual_norm(x, dual)):
            with pytest.raises(kernels.KernelError, match="forward-mode"):
                f()


def test_decay_backward_shape_checks():
    from prometheus_amd.kernels.decay import _DecayResidual

    q, g, s = np.zeros((1, 3, 2, 8), np.float32), np.zeros((1, 3, 2), np.float32), np.zeros((1, 2, 8, 8), np.float32)
    res = _DecayResidual(q, q, q, g, s, 1.0)
    for grads in ((q[:, :2], None), (None, s[:, :1])):
        with pytest.raises(kernels.KernelError):
            kernels.decay_attention_bwd(res, grads)
    with pytest.raises(kernels.KernelError):
        kernels.decay_attention_bwd(_DecayResidual(q, q, q, g, s[:, :1], 1.0), (q, None))


def test_norm_checks():
    x = np.zeros((2, 6), np.float32)
    bad = [
        lambda: kernels.gated_norm(x, x[:1]),
        lambda: kernels.gated_norm(x, x, np.zeros(5)),
        lambda: kernels.gated_norm(x, x, activation="relu"),
        lambda: kernels.gated_norm(x, x, eps=-1.0),
        lambda: kernels.gated_norm(x, x, eps=float("nan")),
        lambda: kernels.gated_norm(x[:, :0], x[:, :0]),
        lambda: kernels.gated_norm(np.zeros((1, 16385)), np.zeros((1, 16385))),
        lambda: kernels.gated_norm(np.float32(1.0), np.float32(1.0)),
        lambda: kernels.residual_norm(x, x[:1]),
        lambda: kernels.residual_norm(x, x, np.zeros(5)),
        lambda: kernels.residual_norm(x, x, post_weight=np.zeros((1, 6))),
        lambda: kernels.residual_norm(x, x, scale=float("inf")),
        lambda: kernels.residual_norm(x, x, eps=-1e-9),
        lambda: kernels.gated_norm_bwd(row_norms._GatedNormResidual(x, x, None, "silu", False, 1e-6, torch.float32), x[:1]),
        lambda: kernels.residual_norm_bwd(row_norms._ResidualNormResidual(x, x, None, None, 1.0, 1e-6), (None, x[:1])),
    ]
    for f in bad:
        with pytest.raises(kernels.KernelError):
            f()


@pytest.mark.parametrize("shape,order", [((3, 4, 5, 8), (0, 1, 2, 3)), ((3, 4, 5, 8), (1, 0, 2, 3)), ((3, 4, 5, 8), (0, 2, 1, 3)),
                                         ((1, 4, 1, 8), (0, 2, 1, 3)), ((6, 8), (0, 1)), ((8,), (0,))])
def test_rows_are_walked_where_they_are(shape, order):
    """Every row's address as the kernels compute it, for views of which some need a copy."""
    base = torch.arange(np.prod(shape)).reshape([shape[i] for i in order]).permute(*np.argsort(order).tolist())
    assert base.shape == shape
    got = row_norms._rows_of(tuple(shape), base.stride(), base.contiguous().stride())
    want = base.reshape(-1, shape[-1])[:, 0].tolist()
    if got is None:
        assert order in ((1, 0, 2, 3), (0, 2, 1, 3))
        return
    rows, inner, st = got
    assert [i // inner * st[0] + i % inner * st[1] for i in range(rows)] == want
    assert [i // inner * st[2] + i % inner * st[3] for i in range(rows)] == [i * shape[-1] for i in range(rows)]


def test_cache_checks():
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0)):
        with pytest.raises(ValueError):
            serving.DecayStateCache(*bad, device="cpu")
    cache = serving.DecayStateCache(1, 3, 2, 8, device="cpu")
    assert cache.pool.shape == (1, 3, 2, 8, 8)
    q, g = torch.zeros(1, 4, 2, 8), torch.zeros(1, 4, 2)
    for f in (lambda: cache.prefill(1, [0], q, q, q, g), lambda: cache.prefill(0, [3], q, q, q, g),
              lambda: cache.prefill(0, [0, 0], q, q, q, g), lambda: cache.prefill(0, [0, 1], q, q, q, g),
              lambda: cache.prefill(0, [0], q[..., :1, :], q[..., :1, :], q[..., :1, :], g[..., :1]),
              lambda: cache.prefill(0, [0], q, q, q, g.requires_grad_(True))):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(RuntimeError, match="host"):
        cache.prefill(0, [0], q, q, q, g.detach())
    with pytest.raises(RuntimeError, match="host"):
        cache.decode(0, torch.zeros(1, dtype=torch.int32), q[:, 0], q[:, 0], q[:, 0], g[:, 0].detach())


# --- the C entry points ---


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_decay_abi_refuses():
    L = _native.lib()

    def fwd(q=P, k=P, v=P, g=P, cu=None, s0=None, slots=None, n_slots=0, o=P, s_out=P, n=1, T=4, Hq=2, H=2, D=8,
            strides=_i64(*[64, 16, 8] * 3), g_sb=8, g_st=2, dt=0, odt=0, scale=1.0, ws=None, nbytes=0):
        return L.pm_decay_attention(q, k, v, g, cu, s0, slots, n_slots, None, None, o, s_out, n, T, Hq, H, D, strides,
                                    g_sb, g_st, dt, odt, scale, ws, nbytes, None)

    E = _native
    odd = ctypes.c_void_p(18)
    for kw, want in ((dict(q=None), E.E_NULL), (dict(g=None), E.E_NULL), (dict(s_out=None), E.E_NULL),
                     (dict(strides=None), E.E_NULL), (dict(n=-1), E.E_SHAPE), (dict(T=-1), E.E_SHAPE),
                     (dict(Hq=3), E.E_SHAPE), (dict(H=0), E.E_SHAPE), (dict(D=0), E.E_SHAPE), (dict(D=257), E.E_SHAPE),
                     (dict(dt=2), E.E_DTYPE), (dict(odt=-1), E.E_DTYPE), (dict(scale=float("inf")), E.E_SHAPE),
                     (dict(strides=_i64(-1, *[64] * 8)), E.E_SHAPE), (dict(g_st=-1), E.E_SHAPE),
                     (dict(strides=_i64(64, (1 << 23) + 1, *[8] * 7)), E.E_SHAPE),
                     (dict(slots=P), E.E_SHAPE), (dict(slots=P, s0=P, n_slots=-1), E.E_SHAPE),
                     (dict(q=odd), E.E_ALIGN), (dict(g=odd), E.E_ALIGN), (dict(n=1 << 20, T=1 << 30), E.E_SHAPE),
                     (dict(cu=P), E.E_WORKSPACE), (dict(T=4096), E.E_WORKSPACE),
                     (dict(T=4096, ws=ctypes.c_void_p(8), nbytes=1 << 30), E.E_WORKSPACE)):
        assert fwd(**kw) == want, kw
    assert fwd(n=0) == 0
    # sizes: none where one workgroup does a sequence, the states of spans otherwise, a table for packed calls
    size = L.pm_decay_attention_workspace_bytes
    assert size(1, 200, 2, 2, 64, 0, 0) == 0 and size(32, 2048, 16, 16, 64, 0, 0) == 0 and size(1, 4096, 2, 2, 64, 0, 0) > 0 and size(3, 10, 2, 2, 64, 1, 0) > 0
    assert size(2, 10, 4, 2, 64, 0, 1) == 2 * 2 * 64 * 64 * 4 and size(1, 4, 3, 2, 8, 0, 0) == 0

    def bwd(q=P, go=P, gq=P, gg=P, gs0=P, s0=None, B=1, T=4, strides=_i64(*[64, 16, 8] * 3), g_sb=8, g_st=2, dt=0, ws=None,
            nbytes=0):
        return L.pm_decay_attention_bwd(q, P, P, P, s0, go, None, gq, P, P, gg, gs0, B, T, 2, 2, 8, strides, g_sb, g_st,
                                        dt, 1.0, ws, nbytes, None)

    for kw, want in ((dict(q=None), E.E_NULL), (dict(go=None), E.E_NULL), (dict(gq=None), E.E_NULL),
                     (dict(B=-1), E.E_SHAPE), (dict(dt=3), E.E_DTYPE), (dict(gg=odd), E.E_ALIGN),
                     (dict(gs0=odd), E.E_ALIGN), (dict(), E.E_WORKSPACE)):
        assert bwd(**kw) == want, kw
    assert bwd(B=0) == 0
    # more workgroups than one launch can have; many short packed sequences are not
    wide = dict(strides=_i64(*[16, 8, 8] * 3), T=1, ws=P, nbytes=1 << 60)
    assert fwd(n=1 << 23, q=odd, **wide) == E.E_SHAPE and fwd(n=1 << 22, q=odd, **wide) == E.E_ALIGN
    assert bwd(B=1 << 22, q=odd, **wide) == E.E_SHAPE and bwd(B=1 << 21, q=odd, **wide) == E.E_ALIGN
    assert size(20000, 1 << 20, 32, 32, 8, 1, 0) > 0 and size(1 << 23, 1 << 23, 2, 2, 8, 1, 0) == 0
    need = L.pm_decay_attention_bwd_workspace_bytes
    assert need(1, 100, 2, 2, 64, 0) == 0 and need(1, 100, 2, 2, 64, 1) > 0 and need(-1, 100, 2, 2, 64, 1) == 0

    def step(s=P, q=P, g=P, o=P, slots=None, n_slots=0, B=1, Hq=2, strides=_i64(*[16, 8] * 3), g_sb=2, dt=0):
        return L.pm_decay_attention_step(s, slots, n_slots, q, P, P, g, o, B, Hq, 2, 8, strides, g_sb, dt, dt, 1.0, None)

    for kw, want in ((dict(s=None), E.E_NULL), (dict(g=None), E.E_NULL), (dict(o=None), E.E_NULL),
                     (dict(strides=None), E.E_NULL), (dict(Hq=5), E.E_SHAPE), (dict(slots=P, n_slots=-1), E.E_SHAPE),
                     (dict(g_sb=-1), E.E_SHAPE), (dict(s=odd), E.E_ALIGN), (dict(dt=7), E.E_DTYPE)):
        assert step(**kw) == want, kw
    assert step(B=0) == 0


def test_norms_abi_refuses():
    L, E = _native.lib(), _native
    odd = ctypes.c_void_p(18)

    def gated(x=P, z=P, w=P, y=P, rows=2, inner=1, C=8, strides=_i64(8, 0, 8, 0), act=0, eps=1e-6, t=0):
        return L.pm_gated_norm(x, z, w, y, rows, inner, C, strides, act, 0, eps, t, 0, 0, 0, None)

    for kw, want in ((dict(x=None), E.E_NULL), (dict(y=None), E.E_NULL), (dict(strides=None), E.E_NULL),
                     (dict(rows=-1), E.E_SHAPE), (dict(inner=0), E.E_SHAPE), (dict(C=0), E.E_SHAPE),
                     (dict(C=16385), E.E_SHAPE), (dict(act=2), E.E_SHAPE), (dict(eps=-1.0), E.E_SHAPE),
                     (dict(eps=float("nan")), E.E_SHAPE), (dict(strides=_i64(8, -1, 8, 0)), E.E_SHAPE),
                     (dict(t=5), E.E_DTYPE), (dict(w=odd), E.E_ALIGN), (dict(y=odd), E.E_ALIGN),
                     (dict(rows=1 << 40), E.E_SHAPE)):
        assert gated(**kw) == want, kw
    assert gated(rows=0) == 0

    def gated_bwd(w=P, gy=P, gx=P, gw=None, ws=None, nbytes=0):
        return L.pm_gated_norm_bwd(P, P, w, gy, gx, P, gw, 2, 1, 8, _i64(8, 0, 8, 0), 0, 0, 1e-6, 0, 0, 0, 0, ws, nbytes, None)

    for kw, want in ((dict(gy=None), E.E_NULL), (dict(gx=None), E.E_NULL), (dict(w=None, gw=P), E.E_NULL),
                     (dict(gw=odd), E.E_ALIGN), (dict(gw=P), E.E_WORKSPACE)):
        assert gated_bwd(**kw) == want, kw

    def res(x=P, r=P, y=P, h=P, rows=2, C=8, st=8, scale=1.0, eps=1e-6, t=0):
        return L.pm_residual_norm(x, r, P, P, y, h, rows, C, st, 8, scale, eps, t, 0, 0, 0, None)

    for kw, want in ((dict(x=None), E.E_NULL), (dict(h=None), E.E_NULL), (dict(rows=-1), E.E_SHAPE), (dict(C=0), E.E_SHAPE),
                     (dict(st=-1), E.E_SHAPE), (dict(scale=float("nan")), E.E_SHAPE), (dict(eps=-1.0), E.E_SHAPE),
                     (dict(t=2), E.E_DTYPE), (dict(r=odd), E.E_ALIGN), (dict(y=odd), E.E_ALIGN)):
        assert res(**kw) == want, kw
    assert res(rows=0) == 0

    def res_bwd(wp=P, gx=P, gw=None, gwp=None):
        return L.pm_residual_norm_bwd(P, P, P, wp, P, P, gx, P, gw, gwp, 2, 8, 8, 8, 1.0, 1e-6, 0, 0, 0, 0, None, 0, None)

    for kw, want in ((dict(gx=None), E.E_NULL), (dict(wp=None, gwp=P), E.E_NULL), (dict(gw=odd), E.E_ALIGN),
                     (dict(gw=P), E.E_WORKSPACE), (dict(gwp=P), E.E_WORKSPACE)):
        assert res_bwd(**kw) == want, kw
    assert L.pm_gated_norm_bwd_workspace_bytes(0, 8) == 0 and L.pm_gated_norm_bwd_workspace_bytes(10, 8) > 0
    assert L.pm_residual_norm_bwd_workspace_bytes(10, 16385) == 0
