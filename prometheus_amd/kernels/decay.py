"""Linear attention with a decay for each head: the matrix-state layer without the delta rule.

Per sequence and key head, with log-decays ``g`` as in ``chunked_gated_delta_rule``::

    S_t = exp(g_t) S_{t-1} + k_t v_t^T,    o_t = scale q_t S_t

A group of query heads may share each key head (and its state). No reference counterpart (the
reference's model has the delta rule only). The arguments follow ``prometheus_amd.kernels``: torch GPU
tensors are used in place, q, k and v as views whose heads' elements are contiguous (parts of one
projection) without a copy; NumPy arrays and CPU tensors are copied over and the results copied back.
bf16 q, k and v stay bf16, anything else is cast to fp32. Outputs have that type unless ``out_dtype``
says otherwise; states and sums are fp32 always.
"""

from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass

import numpy as np
import torch

from prometheus_amd import _native
from prometheus_amd import kernels as _k
from prometheus_amd.kernels import recurrence as _rec

__all__ = [
    "decay_attention",
    "decay_attention_fwd",
    "decay_attention_bwd",
    "decay_attention_varlen",
    "decay_attention_step",
]


_MAX_TOKEN_STRIDE = 1 << 23  # elements


@dataclass(frozen=True)
class _DecayResidual:
    """Residual of ``decay_attention_fwd``: the arrays the kernel consumed (not copied) and the scale."""

    q: _k.Array
    k: _k.Array
    v: _k.Array
    g: _k.Array
    state0: _k.Array
    scale: float


@functools.lru_cache(maxsize=1024)
def _strides(*values):
    """The host array of strides that the kernels read (never written)."""
    return (ctypes.c_int64 * len(values))(*values)


@functools.lru_cache(maxsize=1024)
def _ws_bytes(n_seqs, T, Hq, H, D, packed, in_place) -> int:
    return _native.lib().pm_decay_attention_workspace_bytes(n_seqs, T, Hq, H, D, packed, in_place)


@functools.lru_cache(maxsize=1024)
def _bwd_ws_bytes(B, T, Hq, H, D, gates) -> int:
    return _native.lib().pm_decay_attention_bwd_workspace_bytes(B, T, Hq, H, D, gates)


def _check(q, k, v, g, rank, scale) -> tuple:
    """``(lead, Hq, H, D)`` of a call whose q, k and v have ``rank`` dimensions."""
    qs, ks, vs, gs = _k._shape(q), _k._shape(k), _k._shape(v), _k._shape(g)
    if len(qs) != rank or len(ks) != rank or vs != ks or qs[:-2] != ks[:-2] or qs[-1] != ks[-1]:
        names = {4: "(B, T, heads, D)", 3: "(B, heads, D)"}[rank]
        raise _k.KernelError(f"q, k and v must be {names}, k and v alike and q alike but for its heads; "
                             f"got {qs}, {ks} and {vs}")
    lead, Hq, H, D = qs[:-2], qs[-2], ks[-2], qs[-1]
    if max(qs) >= 2**31:  # (the library's sizes are 32-bit ones: a larger one would come to another there)
        raise _k.KernelError(f"problem too large: {qs}")
    if H < 1 or Hq < 1 or Hq % H:
        raise _k.KernelError(f"q's heads must be a multiple of k's; got {Hq} and {H}")
    if not 1 <= D <= _native.MAX_D:
        raise _k.KernelError(f"head dimension {D} not in [1, {_native.MAX_D}]")
    if gs != (*lead, H) and gs != (H,):
        raise _k.KernelError(f"g shape {gs} is neither {(*lead, H)} nor {(H,)}")
    if not math.isfinite(scale):
        raise _k.KernelError(f"scale must be finite, got {scale}")
    return lead, Hq, H, D


def _check_state(state, want) -> None:
    if state is not None and _k._shape(state) != want:
        raise _k.KernelError(f"state shape {_k._shape(state)} != {want}")


def _out_dtype(out_dtype, dtype):
    return dtype if out_dtype is None else _k._out_dtype(out_dtype)


def _heads(call, x, dtype):
    """``x`` on the call's device in ``dtype``, the elements of a head contiguous (no copy of a view
    that has them so, and its tokens no further apart than the kernels reach)."""
    if isinstance(x, torch.Tensor) and x.dtype == dtype and x.get_device() == call.device.index and (
            x.stride(-1) == 1 or x.shape[-1] <= 1) and x.stride(-3) <= _MAX_TOKEN_STRIDE:
        return x
    return call.dev(x, dtype).contiguous()


def _decays(call, g):
    """``g`` on the call's device in fp32 and its strides but the heads', which are contiguous: zeros
    for one constant a head, and never zeros otherwise."""
    if not (isinstance(g, torch.Tensor) and g.dtype == torch.float32 and g.get_device() == call.device.index):
        g = call.dev(g, torch.float32)
    if g.dim() == 1:
        return g if g.is_contiguous() else g.contiguous(), (0, 0)
    st = g.stride()
    if st[-1] != 1 or 0 in st:
        g = g.contiguous()
    if g.is_contiguous():
        # (a dimension of one element may have any stride)
        H = g.shape[-1]
        return g, ((g.shape[1] * H, H) if g.dim() == 3 else (H, 0))
    return g, (st[:2] if g.dim() == 3 else (st[0], 0))


def _launch(call, qd, kd, vd, gd, g_strides, cu, flag, s0, slots, n_slots, bad, s_out, o, n_seqs, T, scale):
    """The forward on device tensors; o and s_out are written. q, k and v are (n_seqs, T, heads, D), or
    packed (1, T, heads, D) with ``cu``."""
    ptr = _k._ptr
    Hq, H, D = qd.shape[2], kd.shape[2], qd.shape[3]
    in_place = s0 is not None and s0.data_ptr() == s_out.data_ptr()
    nbytes = _ws_bytes(n_seqs, T, Hq, H, D, cu is not None, in_place)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=call.device) if nbytes else None
    _native.check(_native.lib().pm_decay_attention(
        ptr(qd), ptr(kd), ptr(vd), ptr(gd), ptr(cu), ptr(s0), ptr(slots), n_slots, ptr(bad), ptr(flag), ptr(o),
        ptr(s_out), n_seqs, T, Hq, H, D, _strides(*qd.stride()[:3], *kd.stride()[:3], *vd.stride()[:3]), *g_strides,
        _k._code(qd.dtype), _k._code(o.dtype), scale, ptr(ws), nbytes, _k._stream(call.device)))


def _forward(q, k, v, g, state, scale, out_dtype):
    lead, Hq, H, D = _check(q, k, v, g, 4, scale)
    _check_state(state, (lead[0], H, D, D))
    dtype = _k._qkv_dtype(q, k, v)
    odt = _out_dtype(out_dtype, dtype)
    call = _k._Call(q, k, v, g, state)
    with _k._on(call.device):
        qd, kd, vd = _heads(call, q, dtype), _heads(call, k, dtype), _heads(call, v, dtype)
        gd, g_strides = _decays(call, g)
        sd = call.dev(state, torch.float32)
        o = torch.empty((*lead, Hq, D), dtype=odt, device=call.device)
        s_out = torch.empty((lead[0], H, D, D), dtype=torch.float32, device=call.device)
        _launch(call, qd, kd, vd, gd, g_strides, None, None, sd, None, 0, None, s_out, o, lead[0], lead[1], scale)
    return call, (qd, kd, vd, gd, sd), o, s_out


def _launch_bwd(call, tensors, go, gs, scale, want_g, want_state):
    """The backward on device tensors, go in q's type: ``(gq, gk, gv, gg, gstate)``."""
    qd, kd, vd, gd, sd = tensors
    ptr = _k._ptr
    (B, T, Hq, D), H = qd.shape, kd.shape[2]
    gd, g_strides = _decays(call, gd)
    if go is None:
        go = torch.zeros((B, T, Hq, D), dtype=qd.dtype, device=call.device)
    gq, gk, gv = (torch.empty(x.shape, dtype=x.dtype, device=call.device) for x in (qd, kd, vd))
    gg = torch.empty(gd.shape, dtype=torch.float32, device=call.device) if want_g else None
    gs0 = torch.empty((B, H, D, D), dtype=torch.float32, device=call.device) if want_state else None
    nbytes = _bwd_ws_bytes(B, T, Hq, H, D, want_g)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=call.device) if nbytes else None
    _native.check(_native.lib().pm_decay_attention_bwd(
        ptr(qd), ptr(kd), ptr(vd), ptr(gd), ptr(sd), ptr(go), ptr(gs), ptr(gq), ptr(gk), ptr(gv), ptr(gg), ptr(gs0), B,
        T, Hq, H, D, _strides(*qd.stride()[:3], *kd.stride()[:3], *vd.stride()[:3]), *g_strides, _k._code(qd.dtype),
        scale, ptr(ws), nbytes, _k._stream(call.device)))
    return gq, gk, gv, gg, gs0


class _DecayAttention(torch.autograd.Function):
    """``decay_attention`` as a differentiable op; gradients in each input's type."""

    @staticmethod
    def forward(ctx, q, k, v, g, state, scale, out_dtype):
        call, tensors, o, s = _forward(q, k, v, g, state, scale, out_dtype)
        ctx.save_for_backward(*tensors)
        ctx.call, ctx.scale = call, scale
        ctx.saved = [None if t is None else (t.dtype, t.shape, t.stride()) for t in tensors]
        ctx.set_materialize_grads(False)  # a missing gradient is None, not a tensor of zeros
        # (the type and device of each input's gradient, where it is not as the backward gives it)
        ctx.like = None if all(x is d for x, d in zip((q, k, v, g, state), tensors)) else [
            (x.dtype, x.device) if isinstance(x, torch.Tensor) else None for x in (q, k, v, g, state)]
        return call.out(o), call.out(s)

    @staticmethod
    @_k._once
    def backward(ctx, go, gs):
        call, tensors = ctx.call, ctx.saved_tensors
        gpu = call.device.index
        need = ctx.needs_input_grad[:5]
        with _k._on(call.device):
            for t, like in zip(tensors, ctx.saved):
                if t is not None and not ((t.dtype, t.shape, t.stride()) == like and t.get_device() == gpu):
                    # (saved-tensor hooks may hand back another layout, or copies elsewhere or of another type)
                    tensors = [x if x is None else _k._as_saved(x, *like[:2], call.device)
                               for x, like in zip(tensors, ctx.saved)]
                    tensors = [*(_heads(call, x, x.dtype) for x in tensors[:3]), tensors[3],
                               call.dev(tensors[4], torch.float32)]
                    break
            grads = _launch_bwd(call, tensors, call.dev(go, tensors[0].dtype), call.dev(gs, torch.float32), ctx.scale,
                                need[3], need[4])
        if ctx.like is not None:
            grads = [t if t is None or like is None else t.to(device=like[1], dtype=like[0])
                     for t, like in zip(grads, ctx.like)]
        return (*(t if n else None for t, n in zip(grads, need)), None, None)


def decay_attention(q, k, v, g, state=None, *, scale=1.0, out_dtype=None):
    """Linear attention with a decay for each head: ``S_t = exp(g_t) S_{t-1} + k_t v_t^T`` and
    ``o_t = scale q_t S_t``.

    q: (batch, seq, Hq, D), k and v: (batch, seq, H, D), Hq a multiple of H (query head h reads the
    state of key head ``h // (Hq // H)``); D up to 256. g: log-decays (batch, seq, H), or (H,) for one
    constant a head. state: (batch, H, D, D) fp32 initial state, zeros if None. Returns
    ``(o, next_state)``: o shaped like q, in bf16 for bf16 q, k and v and in fp32 otherwise unless
    ``out_dtype`` says so, next_state (batch, H, D, D) fp32.

    fp32 inputs have fp32 accuracy. bf16 inputs enter the products as they are; o and the gradients
    of q, k and v keep 2^-17 of each term before they are rounded to their type, the states and the
    gradients of the decays and of the first state 2^-24. A log-decay below -138 counts as closed.
    Infinities and NaN reach what they reach token by token (an infinity may come out as NaN), in the
    decays' gradient up to 512 tokens more behind theirs.

    Differentiable: when autograd records and a torch input requires grad, the backward is
    ``decay_attention_bwd``.
    """
    if _k._wants_grad(q, k, v, g, state):
        return _DecayAttention.apply(q, k, v, g, state, scale, out_dtype)
    call, _, o, s = _forward(q, k, v, g, state, scale, out_dtype)
    return call.out(o), call.out(s)


def decay_attention_fwd(q, k, v, g, state=None, *, scale=1.0, out_dtype=None):
    """Explicit forward of the VJP pair: ``((o, next_state), residual)`` for ``decay_attention_bwd``."""
    call, tensors, o, s = _forward(q, k, v, g, state, scale, out_dtype)
    kept = (None if t is None else call.out(t) for t in tensors)
    return (call.out(o), call.out(s)), _DecayResidual(*kept, scale)


def decay_attention_bwd(residual: _DecayResidual, grads):
    """Backward of the VJP pair: ``grads = (go, gs)``, dL/do (batch, seq, Hq, D) and dL/dnext_state
    (batch, H, D, D), either may be None. Returns ``(gq, gk, gv, gg, gstate)``: gq, gk and gv in q's
    type, gg shaped like g and gstate in fp32, each as accurate whichever are wanted. With bf16 q, k and
    v an fp32 go is rounded to bf16 first: it is a factor of products, as they are (fp32 q, k and v keep
    it). What heads or tokens share is summed in an order that does not change."""
    go, gs = grads
    r = residual
    lead, Hq, H, D = _check(r.q, r.k, r.v, r.g, 4, r.scale)
    _check_state(r.state0, (lead[0], H, D, D))
    if go is not None and _k._shape(go) != (*lead, Hq, D):
        raise _k.KernelError(f"grad of output shape {_k._shape(go)} != {(*lead, Hq, D)}")
    if gs is not None and _k._shape(gs) != (lead[0], H, D, D):
        raise _k.KernelError(f"grad of state shape {_k._shape(gs)} != {(lead[0], H, D, D)}")
    call = _k._Call(r.q, r.k, r.v, r.g, r.state0, go, gs)
    dtype = _k._qkv_dtype(r.q, r.k, r.v)
    with _k._on(call.device):
        tensors = (*(_heads(call, x, dtype) for x in (r.q, r.k, r.v)), call.dev(r.g, torch.float32),
                   call.dev(r.state0, torch.float32))
        out = _launch_bwd(call, tensors, call.dev(go, dtype), call.dev(gs, torch.float32), r.scale, True, True)
    return tuple(call.out(t) for t in out)


def _packed(q, k, v, g, cu_seqlens, scale):
    """Checks of a packed call: ``(n_tok, Hq, H, D, n_seqs, offsets)``, the offsets as
    ``recurrence._cu`` gives them, and q, k, v and g as (1, N, ..)."""
    qs = _k._shape(q)
    if len(qs) == 3:
        q, k, v = (x[None] for x in (q, k, v))
        g = g if len(_k._shape(g)) == 1 else g[None]
    lead, Hq, H, D = _check(q, k, v, g, 4, scale)
    if lead[0] != 1:
        raise _k.KernelError(f"packed q, k and v must be (N, heads, D) or (1, N, heads, D); got {qs}")
    return lead[1], Hq, H, D, *_rec._cu(cu_seqlens, lead[1]), (q, k, v, g)


def decay_attention_varlen(q, k, v, g, cu_seqlens, state=None, *, scale=1.0, out_dtype=None):
    """Packed batch of independent sequences, the state starting anew at every boundary.

    q, k, v: (N, heads, D) or (1, N, heads, D), g (N, H) or (1, N, H) or (H,); cu_seqlens and its checks
    as ``chunked_delta_rule_varlen``; state: None (zeros) or (n_seqs, H, D, D). Returns
    ``(o, final_states)``, o shaped like q and final_states (n_seqs, H, D, D) fp32 (an empty sequence's
    is its initial state). Forward only: inputs that require grad are refused while autograd records.
    """
    if _k._wants_grad(q, k, v, g, state):
        raise _k.KernelError("decay_attention_varlen is forward only: call it under torch.no_grad()")
    shape = _k._shape(q)
    n_tok, Hq, H, D, n_seqs, cu, (q, k, v, g) = _packed(q, k, v, g, cu_seqlens, scale)
    _check_state(state, (n_seqs, H, D, D))
    dtype = _k._qkv_dtype(q, k, v)
    odt = _out_dtype(out_dtype, dtype)
    call = _k._Call(q, k, v, g, state, cu_seqlens)
    with _k._on(call.device):
        qd, kd, vd = _heads(call, q, dtype), _heads(call, k, dtype), _heads(call, v, dtype)
        gd, g_strides = _decays(call, g)
        sd = call.dev(state, torch.float32)
        o = torch.empty(shape, dtype=odt, device=call.device)
        s_out = torch.empty((n_seqs, H, D, D), dtype=torch.float32, device=call.device)
        cu, flag = _rec._offsets(call, cu, n_seqs, n_tok, 1)
        _launch(call, qd, kd, vd, gd, g_strides, cu, flag, sd, None, 0, None, s_out, o, n_seqs, n_tok, scale)
    return call.out(o), call.out(s_out)


def decay_attention_step(q, k, v, g, state, *, scale=1.0, out_dtype=None):
    """One token: q (B, Hq, D), k and v (B, H, D), g (B, H) or (H,), ``state`` (B, H, D, D) fp32 updated
    in place as in ``delta_rule_step``; returns o (B, Hq, D). fp32 arithmetic. Forward only, as
    ``decay_attention_varlen``."""
    if _k._wants_grad(q, k, v, g, state):
        raise _k.KernelError("decay_attention_step is forward only: call it under torch.no_grad()")
    (batch,), Hq, H, D = _check(q, k, v, g, 3, scale)
    if state is None or _k._shape(state) != (batch, H, D, D):
        raise _k.KernelError(f"state shape {None if state is None else _k._shape(state)} != {(batch, H, D, D)}")
    in_place = isinstance(state, torch.Tensor) and state.device.type == "cuda"
    if in_place and (state.dtype != torch.float32 or not state.is_contiguous()):
        raise _k.KernelError("state must be a contiguous fp32 tensor to be updated in place")
    if not in_place and not isinstance(state, (np.ndarray, torch.Tensor)):
        raise _k.KernelError("state must be an array or tensor to be updated in place")
    if isinstance(state, np.ndarray) and state.dtype != np.float32:
        raise _k.KernelError("state must be fp32 to be updated in place")
    dtype = _k._qkv_dtype(q, k, v)
    odt = _out_dtype(out_dtype, dtype)
    call = _k._Call(q, k, v, g, state)
    with _k._on(call.device):
        qd, kd, vd = _heads(call, q, dtype), _heads(call, k, dtype), _heads(call, v, dtype)
        gd, (g_sb, _) = _decays(call, g)
        sd = state if in_place else call.dev(state, torch.float32)
        o = torch.empty((batch, Hq, D), dtype=odt, device=call.device)
        _step(_k._ptr(sd), None, 0, qd, kd, vd, gd, g_sb, o, scale, _k._stream(call.device))
        if not in_place:
            host = sd.cpu()
            if isinstance(state, np.ndarray):
                state[...] = host.numpy()
            else:
                state.copy_(host)
    return call.out(o)


def _step(state: int | None, slots, n_slots, qd, kd, vd, gd, g_sb, o, scale, stream):
    """One token on device tensors; ``state`` is the states' address."""
    batch, Hq, D = qd.shape
    qs, ks, vs = qd.stride(), kd.stride(), vd.stride()
    _native.check(_native.lib().pm_decay_attention_step(
        state, None if slots is None else slots.data_ptr(), n_slots, qd.data_ptr(), kd.data_ptr(), vd.data_ptr(),
        gd.data_ptr(), o.data_ptr(), batch, Hq, kd.shape[1], D, _strides(qs[0], qs[1], ks[0], ks[1], vs[0], vs[1]), g_sb,
        _k._code(qd.dtype), _k._code(o.dtype), scale, stream))
