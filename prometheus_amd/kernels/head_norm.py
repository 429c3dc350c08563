"""Norms of queries and keys for each head, with the position rotation in the same pass.

What q and k go through between their projection and the delta rule (or any attention): the
model's ``x / max(||x||, 1e-6)`` (``model/__init__.py:203-205``) or an RMS norm, a weight per
dimension, and the rotation of each pair of dimensions by the token's position. One kernel reads
q and k once (in place, as views of a fused projection too) and writes both results. The rotation
and the weights have no reference counterpart.
"""

from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Any

import numpy as np
import torch

from prometheus_amd import _native
from prometheus_amd import kernels as _k

__all__ = ["norm_rotate", "norm_rotate_fwd", "norm_rotate_bwd", "rotation_table"]

_NORMS = {"l2": _native.NORM_L2, "rms": _native.NORM_RMS}


@functools.lru_cache(maxsize=256)
def _strides(*values):
    """The host array of six strides that the kernels read (never written)."""
    return (ctypes.c_int64 * 6)(*values)


@dataclass(frozen=True)
class _NormRotateResidual:
    """Residual of ``norm_rotate_fwd``: the arrays the kernel consumed (not copied) and its options."""

    q: Any
    k: Any
    table: Any
    positions: Any
    q_weight: Any
    k_weight: Any
    norm: str
    eps: float
    interleaved: bool


def rotation_table(n_positions: int, dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """The table ``norm_rotate`` takes: (n_positions, dim) fp32, row p the dim / 2 cosines and
    then the dim / 2 sines of the angles ``p base^(-2 i / dim)``, computed in 64 bits."""
    if n_positions < 0 or dim < 2 or dim % 2:
        raise _k.KernelError(f"rotation_table needs n_positions >= 0 and an even dim >= 2; got {n_positions}, {dim}")
    if device is None:
        device = _k._device()
    rate = torch.exp(torch.arange(0, dim, 2, dtype=torch.float64, device=device) * (-math.log(base) / dim))
    angle = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * rate
    return torch.cat([torch.cos(angle), torch.sin(angle)], 1).float()


def _check(q, k, table, positions, norm, q_weight, k_weight, eps) -> tuple:
    """(B, T, Hq, Hk, D, R, P) of a call; a 3-D q counts as B = 1."""
    qs, ks = _k._shape(q), _k._shape(k)
    if len(qs) not in (3, 4) or len(ks) != len(qs) or ks[:-2] != qs[:-2] or ks[-1] != qs[-1]:
        raise _k.KernelError(f"q and k must be (B, T, H, D) or (N, H, D), alike but for H; got {qs} and {ks}")
    batch, seq = qs[:2] if len(qs) == 4 else (1, qs[0])
    dim = qs[-1]
    if not 1 <= dim <= _native.MAX_D:
        raise _k.KernelError(f"head dimension {dim} not in [1, {_native.MAX_D}]")
    if norm not in _NORMS:
        raise _k.KernelError(f"norm must be one of {sorted(_NORMS)}, got {norm!r}")
    if not eps >= 0.0:
        raise _k.KernelError(f"eps must be >= 0, got {eps}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and _k._shape(w) != (dim,):
            raise _k.KernelError(f"{name} shape {_k._shape(w)} != {(dim,)}")
    rot = rows = 0
    if table is not None:
        ts = _k._shape(table)
        if len(ts) != 2 or ts[1] % 2 or ts[1] > dim:
            raise _k.KernelError(f"table must be (positions, R) with R even and at most {dim}; got {ts}")
        rows, rot = ts
    if positions is not None:
        if table is None:
            raise _k.KernelError("positions need a table")
        if _k._shape(positions) not in ((seq,), qs[:-2]):
            raise _k.KernelError(f"positions shape {_k._shape(positions)} is neither {(seq,)} nor {qs[:-2]}")
        if isinstance(positions, torch.Tensor) and positions.is_cuda:
            if positions.dtype not in (torch.int32, torch.int64):
                raise _k.KernelError(f"positions must be int32 or int64, got {positions.dtype}")
            return batch, seq, qs[-2], ks[-2], dim, rot, rows
        host = np.asarray(positions)
        if not np.issubdtype(host.dtype, np.integer):
            raise _k.KernelError(f"positions must be integers, got {host.dtype}")
        if host.size and (host.min() < 0 or host.max() >= rows):
            raise _k.KernelError(f"positions {host.min()}..{host.max()} outside the table's {rows} rows")
    elif rot and len(qs) == 3:
        raise _k.KernelError("q and k of shape (N, H, D) need positions")
    elif rot and seq > rows:
        raise _k.KernelError(f"{seq} tokens need a table of as many rows; it has {rows}")
    return batch, seq, qs[-2], ks[-2], dim, rot, rows


def _heads(call, x, dtype):
    """``x`` on the call's device in ``dtype``, the elements of a head contiguous."""
    if isinstance(x, torch.Tensor) and x.dtype == dtype and x.get_device() == call.device.index and (
            x.stride(-1) == 1 or x.shape[-1] <= 1):
        return x
    return call.dev(x, dtype)


@functools.lru_cache(maxsize=1024)
def _ws_bytes(B, T, Hq, Hk, D) -> int:
    return _native.lib().pm_norm_rotate_bwd_workspace_bytes(B, T, Hq, Hk, D)


class _Plan:
    """One call's device tensors and the arguments both directions share."""

    def __init__(self, q, k, table, positions, norm, q_weight, k_weight, eps, interleaved, *more):
        self.dims = _check(q, k, table, positions, norm, q_weight, k_weight, eps)
        self.call = call = _k._Call(q, k, table, positions, q_weight, k_weight, *more)
        self.dtype = dtype = _common_bf16(q, k)
        w_dtype = _common_bf16(*(w for w in (q_weight, k_weight) if w is not None))
        self.q, self.k = _heads(call, q, dtype), _heads(call, k, dtype)
        self.wq, self.wk = call.dev(q_weight, w_dtype), call.dev(k_weight, w_dtype)
        self.table = call.dev(table, torch.float32)
        self.pos, pos_sb, pos64 = None, 0, 0
        if positions is not None:
            p = positions if isinstance(positions, torch.Tensor) else torch.from_numpy(np.asarray(positions))
            if p.dtype not in (torch.int32, torch.int64):
                p = p.to(torch.int64)
            if not p.is_cuda:
                p = p.to(call.device)
            if p.dim() == 2 and (p.shape[1] <= 1 or p.stride(1) == 1):
                pos_sb = p.stride(0)
            elif not p.is_contiguous():
                p = p.contiguous()
                pos_sb = p.shape[1] if p.dim() == 2 else 0
            self.pos, pos64 = p, int(p.dtype == torch.int64)
        qs, ks = self.q.stride(), self.k.stride()
        if len(qs) == 3:
            qs, ks = (0, *qs), (0, *ks)
        self.shared = (*self.dims, _strides(*qs[:3], *ks[:3]), pos_sb, pos64, _NORMS[norm], eps, int(interleaved),
                       _k._code(dtype), _k._code(w_dtype))

    def tensors(self):
        return self.q, self.k, self.table, self.pos, self.wq, self.wk


def _common_bf16(*xs) -> torch.dtype:
    """bf16 if there are arrays and all are bf16 tensors, else fp32."""
    for x in xs:
        if not isinstance(x, torch.Tensor) or x.dtype != torch.bfloat16:
            return torch.float32
    return torch.bfloat16 if xs else torch.float32


def _forward(q, k, table, positions, norm, q_weight, k_weight, eps, interleaved):
    # (the plan's shape checks come first; its _Call then finds the device)
    plan = _Plan(q, k, table, positions, norm, q_weight, k_weight, eps, interleaved)
    dev, ptr = plan.call.device, _k._ptr
    with _k._on(dev):
        qo = torch.empty_like(plan.q, memory_format=torch.contiguous_format)
        ko = torch.empty_like(plan.k, memory_format=torch.contiguous_format)
        _native.check(_native.lib().pm_norm_rotate(
            ptr(plan.q), ptr(plan.k), ptr(plan.table), ptr(plan.pos), ptr(plan.wq), ptr(plan.wk), ptr(qo), ptr(ko),
            *plan.shared, _k._stream(dev)))
    return plan, qo, ko


def _launch_bwd(dev, tensors, shared, gqo, gko, want_weights):
    """The backward on device tensors: ``(gq, gk, gq_weight, gk_weight)``."""
    q, k, table, pos, wq, wk = tensors
    L, ptr, f32 = _native.lib(), _k._ptr, torch.float32
    gq = torch.empty_like(q, memory_format=torch.contiguous_format)
    gk = torch.empty_like(k, memory_format=torch.contiguous_format)
    gwq, gwk = (torch.empty(w.shape, dtype=f32, device=dev) if w is not None and want else None
                for w, want in zip((wq, wk), want_weights))
    nbytes = _ws_bytes(*shared[:5]) if gwq is not None or gwk is not None else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _native.check(L.pm_norm_rotate_bwd(
        ptr(q), ptr(k), ptr(table), ptr(pos), ptr(wq), ptr(wk), ptr(gqo), ptr(gko), ptr(gq), ptr(gk), ptr(gwq),
        ptr(gwk), *shared, ptr(ws), nbytes, _k._stream(dev)))
    return gq, gk, gwq, gwk


class _NormRotate(torch.autograd.Function):
    """``norm_rotate`` as a differentiable op; gradients in each input's type."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, table, positions, norm, eps, interleaved):
        plan, qo, ko = _forward(q, k, table, positions, norm, q_weight, k_weight, eps, interleaved)
        tensors = plan.tensors()
        ctx.save_for_backward(*tensors)
        ctx.call, ctx.options = plan.call, (norm, eps, interleaved)
        ctx.shared = plan.shared
        ctx.saved = [None if t is None else (t.dtype, t.shape, t.stride()) for t in tensors]
        ctx.set_materialize_grads(False)  # a missing gradient is None, not a tensor of zeros
        # (the type and device of each input's gradient, where it is not as the backward gives it)
        as_given = q is plan.q and k is plan.k and all(
            w is None or (w is u and w.dtype == torch.float32) for w, u in ((q_weight, plan.wq), (k_weight, plan.wk)))
        ctx.like = None if as_given else [(t.dtype, t.device) if isinstance(t, torch.Tensor) else None
                                          for t in (q, k, q_weight, k_weight)]
        return plan.call.out(qo), plan.call.out(ko)

    @staticmethod
    @_k._once
    def backward(ctx, gq, gk):
        tensors, need = ctx.saved_tensors, ctx.needs_input_grad
        want = (need[2], need[3])
        call, gpu = ctx.call, ctx.call.device.index
        for t, like in zip(tensors, ctx.saved):
            if t is not None and not ((t.dtype, t.shape, t.stride()) == like and t.get_device() == gpu):
                # (saved-tensor hooks may hand back another layout, or copies elsewhere or of another type)
                tensors = [u if u is None else _k._as_saved(u, *like[:2], call.device)
                           for u, like in zip(tensors, ctx.saved)]
                grads = _backward(_NormRotateResidual(*tensors, *ctx.options), (gq, gk), want)
                break
        else:
            with _k._on(call.device):
                grads = _launch_bwd(call.device, tensors, ctx.shared, call.dev(gq), call.dev(gk), want)
        if ctx.like is not None:
            grads = [t if t is None or like is None else t.to(device=like[1], dtype=like[0])
                     for t, like in zip(grads, ctx.like)]
        return (*[t if n else None for t, n in zip(grads, need)], None, None, None, None, None)


def norm_rotate(q, k, table=None, positions=None, *, norm="l2", q_weight=None, k_weight=None, eps=1e-6,
                interleaved=False):
    """Each head of q and k normalised, weighted and rotated; returns ``(q', k')``.

    q: (B, T, Hq, D) or (N, Hq, D), k alike with its own number of heads; D up to 256; any strides
    with the elements of a head contiguous are read in place. ``norm``: "l2" is
    ``x / max(||x||, eps)`` (what the delta rule wants of its keys), "rms"
    ``x / sqrt(mean(x^2) + eps)``. q_weight, k_weight: (D,) or None.

    table: None (no rotation) or (P, R) fp32 from ``rotation_table``: the first R dimensions are
    turned in pairs (i, i + R / 2), or (2 i, 2 i + 1) with ``interleaved``. positions: integers of
    shape (T,), (B, T) or (N,), each token's row of the table; None counts 0, 1, 2, ... in every
    batch row. Positions on the host are checked here; for those on the GPU, which are not copied
    back, a token outside the table comes out as NaN and nothing outside the table is read.

    bf16 q and k give bf16 results, anything else fp32; arithmetic is fp32 with one rounding at
    the end. Differentiable in q, k and the weights; a table that requires grad is refused while
    autograd records.
    """
    if _k._wants_grad(table):
        raise _k.KernelError("norm_rotate has no gradient of the table: detach it")
    if _k._wants_grad(q, k, q_weight, k_weight):
        return _NormRotate.apply(q, k, q_weight, k_weight, table, positions, norm, eps, interleaved)
    plan, qo, ko = _forward(q, k, table, positions, norm, q_weight, k_weight, eps, interleaved)
    return plan.call.out(qo), plan.call.out(ko)


def norm_rotate_fwd(q, k, table=None, positions=None, *, norm="l2", q_weight=None, k_weight=None, eps=1e-6,
                    interleaved=False):
    """Explicit forward of the VJP pair: ``((q', k'), residual)`` for ``norm_rotate_bwd``."""
    plan, qo, ko = _forward(q, k, table, positions, norm, q_weight, k_weight, eps, interleaved)
    back = plan.call.out
    kept = (None if t is None else back(t) for t in (plan.q, plan.k, plan.table, plan.pos, plan.wq, plan.wk))
    return (back(qo), back(ko)), _NormRotateResidual(*kept, norm, eps, interleaved)


def norm_rotate_bwd(residual: _NormRotateResidual, grads):
    """Backward of the VJP pair: ``grads = (gq', gk')``, shaped like the outputs, either may be
    None. Returns ``(gq, gk, gq_weight, gk_weight)``: q's and k's in their type, the weights' in
    fp32 (None where there is no weight), summed in an order that does not change."""
    return _backward(residual, grads, (True, True))


def _backward(res, grads, want_weights):
    for name, x, gx in (("q", res.q, grads[0]), ("k", res.k, grads[1])):
        if gx is not None and _k._shape(gx) != _k._shape(x):
            raise _k.KernelError(f"grad of {name} shape {_k._shape(gx)} != {_k._shape(x)}")
    plan = _Plan(res.q, res.k, res.table, res.positions, res.norm, res.q_weight, res.k_weight, res.eps,
                 res.interleaved, *grads)
    call = plan.call
    with _k._on(call.device):
        gqo, gko = (call.dev(x, plan.dtype) for x in grads)
        out = _launch_bwd(call.device, plan.tensors(), plan.shared, gqo, gko, want_weights)
    return tuple(None if t is None else call.out(t) for t in out)
