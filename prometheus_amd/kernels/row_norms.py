"""The norms around a layer: with its gate before the output projection, and between two blocks.

``gated_norm`` normalises the rows of a layer's output (its heads, or its whole width), weights them
and multiplies them by the activated gate. ``residual_norm`` ends a block and begins the next: the
norm of the block's output (where it has one), the sum with the residual, and the norm of that. No
reference counterpart. The arguments follow ``prometheus_amd.kernels``; rows are read in place through
strides, bf16 tensors stay bf16, anything else is cast to fp32; arithmetic is fp32 with one rounding at
the end, and the weights' gradients are fp32, summed in an order that does not change.
"""

from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Any

import torch

from prometheus_amd import _native
from prometheus_amd import kernels as _k

__all__ = ["gated_norm", "gated_norm_fwd", "gated_norm_bwd", "residual_norm", "residual_norm_fwd", "residual_norm_bwd"]

_ACTIVATIONS = {"silu": _native.ACT_SILU, "sigmoid": _native.ACT_SIGMOID}


@dataclass(frozen=True)
class _GatedNormResidual:
    """Residual of ``gated_norm_fwd``: the arrays the kernel consumed (not copied) and its options."""

    x: Any
    gate: Any
    weight: Any
    activation: str
    gate_first: bool
    eps: float
    y_dtype: torch.dtype


@dataclass(frozen=True)
class _ResidualNormResidual:
    """Residual of ``residual_norm_fwd``: the arrays the kernel consumed (not copied) and its options."""

    x: Any
    residual: Any
    weight: Any
    post_weight: Any
    scale: float
    eps: float


def _dtype(x) -> torch.dtype:
    return torch.bfloat16 if isinstance(x, torch.Tensor) and x.dtype == torch.bfloat16 else torch.float32


def _even(shape, strides):
    """The stride between consecutive ones of the elements that ``shape`` and ``strides`` enumerate,
    or None where they are not evenly spaced."""
    if 0 in shape:
        return 0
    step, reach = None, 0
    for size, stride in zip(reversed(shape), reversed(strides)):
        if size == 1:
            continue
        if step is None:
            step = stride
        elif stride != reach:
            return None
        reach = stride * size
    return 0 if step is None else step


@functools.lru_cache(maxsize=1024)
def _rows_of(shape, x_strides, z_strides):
    """``(rows, inner, strides array)`` that walk the rows of both tensors, or None where one of them
    has to be copied: rows evenly spaced, or evenly spaced groups of the last dimension but one."""
    lead = shape[:-1]
    rows = math.prod(lead)
    if rows == 0:
        return 0, 1, (ctypes.c_int64 * 4)(0, 0, 0, 0)
    both = (x_strides[:-1], z_strides[:-1])
    whole = [_even(lead, s) for s in both]
    if None not in whole:
        return rows, 1, (ctypes.c_int64 * 4)(whole[0], 0, whole[1], 0)
    outer = [_even(lead[:-1], s[:-1]) for s in both]
    if None in outer or lead[-1] >= 2**31:  # (the library counts a group's rows in 32 bits)
        return None
    return rows, lead[-1], (ctypes.c_int64 * 4)(outer[0], both[0][-1], outer[1], both[1][-1])


def _dev(call, x, dtype):
    """``x`` on the call's device in ``dtype``, the elements of a row contiguous."""
    if isinstance(x, torch.Tensor) and x.dtype == dtype and x.get_device() == call.device.index and (
            x.stride(-1) == 1 or x.shape[-1] <= 1):
        return x
    return call.dev(x, dtype)


class _Quick:
    """Stands for the ``_Call`` of tensors that are all on one GPU as the kernels take them."""

    host_numpy = host_torch = False

    def __init__(self, device):
        self.device = device

    dev = _k._Call.dev

    @staticmethod
    def out(t):
        return t


_CODES = {torch.float32: _native.DTYPE_F32, torch.bfloat16: _native.DTYPE_BF16}
_QUICK: dict = {}


def _quick(shape, rows, weights):
    """A ``_Quick`` where every one of the tensors ``rows`` has this shape, and every one of ``weights``
    (or None) its last dimension's, all contiguous, fp32 or bf16 and on one GPU, so that no other check of
    shapes, types or devices is left to do; None where that is not so."""
    gpu = -1
    for x in rows:
        if not (isinstance(x, torch.Tensor) and x.shape == shape and x.dtype in _CODES and x.is_contiguous()):
            return None
        at = x.get_device()
        if at < 0 or (gpu >= 0 and at != gpu):
            return None
        gpu = at
    for w in weights:
        if w is not None and not (isinstance(w, torch.Tensor) and w.dim() == 1 and w.shape[0] == shape[-1]
                                  and w.dtype in _CODES and w.is_contiguous() and w.get_device() == gpu):
            return None
    call = _QUICK.get(gpu)
    if call is None:
        call = _QUICK[gpu] = _Quick(torch.device("cuda", gpu))
    return call


def _width(shape, *weights) -> int:
    if not shape or not 1 <= shape[-1] <= _native.NORM_MAX_ROW:
        raise _k.KernelError(f"rows must have 1 to {_native.NORM_MAX_ROW} elements; got shape {shape}")
    for name, w in weights:
        if w is not None and _k._shape(w) != (shape[-1],):
            raise _k.KernelError(f"{name} shape {_k._shape(w)} != {(shape[-1],)}")
    return shape[-1]


def _check_eps(eps) -> None:
    if not eps >= 0.0:
        raise _k.KernelError(f"eps must be >= 0, got {eps}")


@functools.lru_cache(maxsize=64)
def _one_stride(width):
    return (ctypes.c_int64 * 4)(width, 0, width, 0)


class _GatedPlan:
    """One call's device tensors and the arguments both directions share."""

    def __init__(self, x, gate, weight, activation, gate_first, eps, y_dtype, *more):
        if activation not in _ACTIVATIONS:
            raise _k.KernelError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
        _check_eps(eps)
        shape = _k._shape(x)
        call = _quick(shape, (x, gate), (weight,)) if shape and 0 < shape[-1] <= _native.NORM_MAX_ROW and not more else None
        if call is not None:
            self.call, self.x, self.gate, self.weight = call, x, gate, weight
            self.rows, self.width = x.numel() // shape[-1], shape[-1]
            self.y_dtype = x.dtype if y_dtype is None else _k._out_dtype(y_dtype)
            self.shared = (self.rows, 1, self.width, _one_stride(self.width), _ACTIVATIONS[activation], int(gate_first),
                           eps, _CODES[x.dtype], _CODES[gate.dtype], _CODES[self.y_dtype],
                           0 if weight is None else _CODES[weight.dtype])
            return
        width = _width(shape, ("weight", weight))
        if _k._shape(gate) != shape:
            raise _k.KernelError(f"gate shape {_k._shape(gate)} != {shape}")
        self.call = call = _k._Call(x, gate, weight, *more)
        xt, zt, wt = _dtype(x), _dtype(gate), _dtype(weight)
        self.y_dtype = xt if y_dtype is None else _k._out_dtype(y_dtype)
        xd, zd = _dev(call, x, xt), _dev(call, gate, zt)
        rows = _rows_of(shape, xd.stride(), zd.stride())
        if rows is None:
            xd, zd = xd.contiguous(), zd.contiguous()
            rows = _rows_of(shape, xd.stride(), zd.stride())
        self.x, self.gate, self.weight = xd, zd, call.dev(weight, wt)
        self.rows, inner, strides = rows
        self.width = width
        self.shared = (self.rows, inner, width, strides, _ACTIVATIONS[activation], int(gate_first), eps, _k._code(xt),
                       _k._code(zt), _k._code(self.y_dtype), _k._code(wt))


@functools.lru_cache(maxsize=1024)
def _gated_ws_bytes(rows, C) -> int:
    return _native.lib().pm_gated_norm_bwd_workspace_bytes(rows, C)


def _gated_forward(x, gate, weight, activation, gate_first, eps, out_dtype):
    plan = _GatedPlan(x, gate, weight, activation, gate_first, eps, out_dtype)
    dev, ptr = plan.call.device, _k._ptr
    with _k._on(dev):
        y = torch.empty_like(plan.x, dtype=plan.y_dtype, memory_format=torch.contiguous_format)
        _native.check(_native.lib().pm_gated_norm(plan.x.data_ptr(), plan.gate.data_ptr(), ptr(plan.weight), y.data_ptr(),
                                                  *plan.shared, _k._stream(dev)))
    return plan, y


def _gated_launch_bwd(dev, tensors, shared, gy, want_weight):
    """The backward on device tensors: ``(gx, g_gate, g_weight)``."""
    x, gate, weight = tensors
    ptr = _k._ptr
    gx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    gz = torch.empty(x.shape, dtype=gate.dtype, device=dev)
    gw = torch.empty(weight.shape, dtype=torch.float32, device=dev) if weight is not None and want_weight else None
    nbytes = _gated_ws_bytes(shared[0], shared[2]) if gw is not None else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _native.check(_native.lib().pm_gated_norm_bwd(ptr(x), ptr(gate), ptr(weight), ptr(gy), ptr(gx), ptr(gz), ptr(gw),
                                                  *shared, ptr(ws), nbytes, _k._stream(dev)))
    return gx, gz, gw


def _same(tensors, saved, gpu) -> bool:
    """Whether autograd handed the saved tensors back as they were (its hooks may give another layout,
    or copies elsewhere or of another type)."""
    return all(t is None or ((t.dtype, t.shape, t.stride()) == like and t.get_device() == gpu)
               for t, like in zip(tensors, saved))


def _layouts(tensors):
    return [None if t is None else (t.dtype, t.shape, t.stride()) for t in tensors]


def _like(inputs, tensors, n_weights):
    """The type and device of each input's gradient, or None where the backward gives them so: the
    input itself was used, and a weight (the last ``n_weights``) is fp32."""
    first = len(inputs) - n_weights
    if all(x is d and (i < first or x is None or x.dtype == torch.float32)
           for i, (x, d) in enumerate(zip(inputs, tensors))):
        return None
    return [(x.dtype, x.device) if isinstance(x, torch.Tensor) else None for x in inputs]


def _as_inputs(grads, like, need):
    if like is not None:
        grads = [g if g is None or t is None else g.to(device=t[1], dtype=t[0]) for g, t in zip(grads, like)]
    return [g if n else None for g, n in zip(grads, need)]


class _GatedNorm(torch.autograd.Function):
    """``gated_norm`` as a differentiable op; gradients in each input's type."""

    @staticmethod
    def forward(ctx, x, gate, weight, activation, gate_first, eps, out_dtype):
        plan, y = _gated_forward(x, gate, weight, activation, gate_first, eps, out_dtype)
        tensors = (plan.x, plan.gate, plan.weight)
        ctx.save_for_backward(*tensors)
        ctx.call, ctx.shared, ctx.options = plan.call, plan.shared, (activation, gate_first, eps, plan.y_dtype)
        ctx.saved = _layouts(tensors)
        ctx.like = _like((x, gate, weight), tensors, 1)
        return plan.call.out(y)

    @staticmethod
    @_k._once
    def backward(ctx, gy):
        tensors, need, call = ctx.saved_tensors, ctx.needs_input_grad, ctx.call
        if _same(tensors, ctx.saved, call.device.index):
            with _k._on(call.device):
                grads = _gated_launch_bwd(call.device, tensors, ctx.shared, call.dev(gy, ctx.options[3]), need[2])
        else:
            tensors = [t if t is None else _k._as_saved(t, *s[:2], call.device) for t, s in zip(tensors, ctx.saved)]
            grads = _gated_backward(_GatedNormResidual(*tensors, *ctx.options), gy, need[2])
        return (*_as_inputs(grads, ctx.like, need), None, None, None, None)


def gated_norm(x, gate, weight=None, *, activation="silu", gate_first=False, eps=1e-6, out_dtype=None):
    """The rows of x normalised, weighted and gated: ``x / sqrt(mean(x^2) + eps) weight act(gate)``.

    x, gate: the same shape (..., C), C up to 16384 (the heads of a layer's output, or its whole
    width); strides with the elements of a row contiguous are read in place. weight: (C,) or None.
    ``activation``: "silu" (``z sigmoid(z)``) or "sigmoid". ``gate_first``: the gate comes before the
    norm, ``u / sqrt(mean(u^2) + eps) weight`` of ``u = x act(gate)``. Returns a tensor shaped like x,
    in its type (bf16 or fp32) unless ``out_dtype`` says otherwise. Differentiable in x, the gate and
    the weight (or ``gated_norm_fwd`` / ``_bwd``).
    """
    if _k._wants_grad(x, gate, weight):
        return _GatedNorm.apply(x, gate, weight, activation, gate_first, eps, out_dtype)
    plan, y = _gated_forward(x, gate, weight, activation, gate_first, eps, out_dtype)
    return plan.call.out(y)


def gated_norm_fwd(x, gate, weight=None, *, activation="silu", gate_first=False, eps=1e-6, out_dtype=None):
    """Explicit forward of the VJP pair: ``(y, residual)`` for ``gated_norm_bwd``."""
    plan, y = _gated_forward(x, gate, weight, activation, gate_first, eps, out_dtype)
    kept = (None if t is None else plan.call.out(t) for t in (plan.x, plan.gate, plan.weight))
    return plan.call.out(y), _GatedNormResidual(*kept, activation, gate_first, eps, plan.y_dtype)


def gated_norm_bwd(residual: _GatedNormResidual, gy):
    """Backward of the VJP pair: gy shaped like y. Returns ``(gx, g_gate, g_weight)``, in x's and the
    gate's type and fp32 (None without a weight)."""
    return _gated_backward(residual, gy, True)


def _gated_backward(res, gy, want_weight):
    if _k._shape(gy) != _k._shape(res.x):
        raise _k.KernelError(f"grad of output shape {_k._shape(gy)} != {_k._shape(res.x)}")
    plan = _GatedPlan(res.x, res.gate, res.weight, res.activation, res.gate_first, res.eps, res.y_dtype, gy)
    call = plan.call
    with _k._on(call.device):
        out = _gated_launch_bwd(call.device, (plan.x, plan.gate, plan.weight), plan.shared, call.dev(gy, plan.y_dtype),
                                want_weight)
    return tuple(None if t is None else call.out(t) for t in out)


class _ResidualPlan:
    """One call's device tensors and the arguments both directions share."""

    def __init__(self, x, residual, weight, post_weight, scale, eps, *more):
        if not math.isfinite(scale):
            raise _k.KernelError(f"scale must be finite, got {scale}")
        _check_eps(eps)
        shape = _k._shape(x)
        call = (_quick(shape, (x, residual), (weight, post_weight))
                if shape and 0 < shape[-1] <= _native.NORM_MAX_ROW and not more else None)
        if call is not None:
            self.call, self.x, self.residual, self.weight, self.post_weight = call, x, residual, weight, post_weight
            width = shape[-1]
            self.shared = (x.numel() // width, width, width, width, scale, eps, _CODES[x.dtype], _CODES[residual.dtype],
                           0 if weight is None else _CODES[weight.dtype],
                           0 if post_weight is None else _CODES[post_weight.dtype])
            return
        width = _width(shape, ("weight", weight), ("post_weight", post_weight))
        if _k._shape(residual) != shape:
            raise _k.KernelError(f"residual shape {_k._shape(residual)} != {shape}")
        self.call = call = _k._Call(x, residual, weight, post_weight, *more)
        xt, rt, wt, pt = (_dtype(t) for t in (x, residual, weight, post_weight))
        xd, rd = _dev(call, x, xt), _dev(call, residual, rt)
        x_st, r_st = _even(shape[:-1], xd.stride()[:-1]), _even(shape[:-1], rd.stride()[:-1])
        if x_st is None:
            xd, x_st = xd.contiguous(), width
        if r_st is None:
            rd, r_st = rd.contiguous(), width
        self.x, self.residual = xd, rd
        self.weight, self.post_weight = call.dev(weight, wt), call.dev(post_weight, pt)
        self.shared = (math.prod(shape[:-1]), width, x_st, r_st, scale, eps, _k._code(xt), _k._code(rt), _k._code(wt),
                       _k._code(pt))

    def tensors(self):
        return self.x, self.residual, self.weight, self.post_weight


@functools.lru_cache(maxsize=1024)
def _residual_ws_bytes(rows, C) -> int:
    return _native.lib().pm_residual_norm_bwd_workspace_bytes(rows, C)


def _residual_forward(x, residual, weight, post_weight, scale, eps):
    plan = _ResidualPlan(x, residual, weight, post_weight, scale, eps)
    dev, ptr = plan.call.device, _k._ptr
    with _k._on(dev):
        y = torch.empty_like(plan.x, memory_format=torch.contiguous_format)
        h = torch.empty_like(plan.residual, memory_format=torch.contiguous_format)
        _native.check(_native.lib().pm_residual_norm(
            plan.x.data_ptr(), plan.residual.data_ptr(), ptr(plan.weight), ptr(plan.post_weight), y.data_ptr(),
            h.data_ptr(), *plan.shared, _k._stream(dev)))
    return plan, y, h


def _residual_launch_bwd(dev, tensors, shared, gy, gh, want_weights):
    """The backward on device tensors: ``(gx, g_residual, g_weight, g_post_weight)``."""
    x, residual, *weights = tensors
    ptr = _k._ptr
    gx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    gr = torch.empty(x.shape, dtype=residual.dtype, device=dev)
    gw, gwp = (torch.empty(w.shape, dtype=torch.float32, device=dev) if w is not None and want else None
               for w, want in zip(weights, want_weights))
    nbytes = _residual_ws_bytes(*shared[:2]) if gw is not None or gwp is not None else 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _native.check(_native.lib().pm_residual_norm_bwd(
        *(ptr(t) for t in tensors), ptr(gy), ptr(gh), ptr(gx), ptr(gr), ptr(gw), ptr(gwp), *shared, ptr(ws), nbytes,
        _k._stream(dev)))
    return gx, gr, gw, gwp


class _ResidualNorm(torch.autograd.Function):
    """``residual_norm`` as a differentiable op; gradients in each input's type."""

    @staticmethod
    def forward(ctx, x, residual, weight, post_weight, scale, eps):
        plan, y, h = _residual_forward(x, residual, weight, post_weight, scale, eps)
        tensors = plan.tensors()
        ctx.save_for_backward(*tensors)
        ctx.call, ctx.shared, ctx.options = plan.call, plan.shared, (scale, eps)
        ctx.saved = _layouts(tensors)
        ctx.set_materialize_grads(False)  # a missing gradient is None, not a tensor of zeros
        ctx.like = _like((x, residual, weight, post_weight), tensors, 2)
        return plan.call.out(y), plan.call.out(h)

    @staticmethod
    @_k._once
    def backward(ctx, gy, gh):
        tensors, need, call = ctx.saved_tensors, ctx.needs_input_grad, ctx.call
        if _same(tensors, ctx.saved, call.device.index):
            with _k._on(call.device):
                grads = _residual_launch_bwd(call.device, tensors, ctx.shared, call.dev(gy, ctx.saved[0][0]),
                                             call.dev(gh, ctx.saved[1][0]), need[2:4])
        else:
            tensors = [t if t is None else _k._as_saved(t, *s[:2], call.device) for t, s in zip(tensors, ctx.saved)]
            grads = _residual_backward(_ResidualNormResidual(*tensors, *ctx.options), (gy, gh), need[2:4])
        return (*_as_inputs(grads, ctx.like, need), None, None)


def residual_norm(x, residual, weight=None, *, post_weight=None, scale=1.0, eps=1e-6):
    """The end of a block and the beginning of the next: ``h = residual + scale b`` and
    ``y = h / sqrt(mean(h^2) + eps) weight``, b the block's output x, or with a ``post_weight`` its norm
    ``x / sqrt(mean(x^2) + eps) post_weight``. Returns ``(y, h)``.

    x, residual: the same shape (..., C), C up to 16384; evenly spaced rows are read in place. weight,
    post_weight: (C,) or None. y has x's type, h the residual's (bf16 or fp32 each); y is computed from
    h before its rounding. Differentiable in x, the residual and the weights (or ``residual_norm_fwd`` /
    ``_bwd``).
    """
    if _k._wants_grad(x, residual, weight, post_weight):
        return _ResidualNorm.apply(x, residual, weight, post_weight, scale, eps)
    plan, y, h = _residual_forward(x, residual, weight, post_weight, scale, eps)
    return plan.call.out(y), plan.call.out(h)


def residual_norm_fwd(x, residual, weight=None, *, post_weight=None, scale=1.0, eps=1e-6):
    """Explicit forward of the VJP pair: ``((y, h), residual)`` for ``residual_norm_bwd``."""
    plan, y, h = _residual_forward(x, residual, weight, post_weight, scale, eps)
    kept = (None if t is None else plan.call.out(t) for t in plan.tensors())
    return (plan.call.out(y), plan.call.out(h)), _ResidualNormResidual(*kept, scale, eps)


def residual_norm_bwd(residual: _ResidualNormResidual, grads):
    """Backward of the VJP pair: ``grads = (gy, gh)``, shaped like x, either may be None. Returns
    ``(gx, g_residual, g_weight, g_post_weight)``, in x's and the residual's type and fp32 (None where
    there is no weight)."""
    return _residual_backward(residual, grads, (True, True))


def _residual_backward(res, grads, want_weights):
    for name, g in zip(("y", "h"), grads):
        if g is not None and _k._shape(g) != _k._shape(res.x):
            raise _k.KernelError(f"grad of {name} shape {_k._shape(g)} != {_k._shape(res.x)}")
    plan = _ResidualPlan(res.x, res.residual, res.weight, res.post_weight, res.scale, res.eps, *grads)
    call = plan.call
    with _k._on(call.device):
        out = _residual_launch_bwd(call.device, plan.tensors(), plan.shared, call.dev(grads[0], plan.x.dtype),
                                   call.dev(grads[1], plan.residual.dtype), want_weights)
    return tuple(None if t is None else call.out(t) for t in out)
