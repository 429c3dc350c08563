"""The elementwise gated linear recurrence: the vector-state layer beside the delta rule.

Per sequence and channel, with log-gates ``g`` as in ``chunked_kda_rule``::

    h_t = exp(g_t) h_{t-1} + x_t

No reference counterpart (the reference's model has matrix states only). The arguments follow
``prometheus_amd.kernels``: torch GPU tensors are used in place, x and g as views whose channels
are contiguous (the halves of one projection) without a copy; NumPy arrays and CPU tensors are
copied over and the results copied back. bf16 x stays bf16 and then takes bf16 or fp32 gates;
every other type is cast to fp32. Outputs are fp32 unless ``out_dtype`` asks for bf16; states
and sums are fp32 always.
"""

from __future__ import annotations

import functools
from dataclasses import dataclass

import numpy as np
import torch

from prometheus_amd import _native
from prometheus_amd import kernels as _k

__all__ = [
    "linear_recurrence",
    "linear_recurrence_fwd",
    "linear_recurrence_bwd",
    "linear_recurrence_varlen",
    "linear_recurrence_step",
]


@dataclass(frozen=True)
class _RecurrenceResidual:
    """Residual of ``linear_recurrence_fwd``: ``x`` and ``g`` as the kernel consumed them (not
    copied), the states before every ``PM_RECURRENCE_SPAN`` tokens ``kept``, and h's type."""

    x: _k.Array
    g: _k.Array
    kept: _k.Array
    h_dtype: torch.dtype


def _types(x, g) -> tuple[torch.dtype, torch.dtype]:
    bf16 = torch.bfloat16
    xt = bf16 if isinstance(x, torch.Tensor) and x.dtype == bf16 else torch.float32
    gt = bf16 if xt == bf16 and isinstance(g, torch.Tensor) and g.dtype == bf16 else torch.float32
    return xt, gt


def _rows(call, x, dtype):
    """``x`` on the call's device in ``dtype``, its last dimension contiguous (no copy of a view
    that has it so)."""
    if isinstance(x, torch.Tensor) and x.dtype == dtype and x.get_device() == call.device.index and (
            x.stride(-1) == 1 or x.shape[-1] <= 1):
        return x
    return call.dev(x, dtype)


def _check(x, g, state, rank) -> tuple:
    xs, gs = _k._shape(x), _k._shape(g)
    if len(xs) != rank or gs != xs:
        names = {3: "(B, T, C)", 2: "(B, C)"}[rank]
        raise _k.KernelError(f"x and g must both have shape {names}; got {xs} and {gs}")
    if state is not None and _k._shape(state) != (xs[0], xs[-1]):
        raise _k.KernelError(f"state shape {_k._shape(state)} != {(xs[0], xs[-1])}")
    return xs


@functools.lru_cache(maxsize=1024)
def _ws_bytes(n_seqs, T, C, packed, x_code) -> int:
    """Bytes of the forward's workspace and (packed False) of the backward's."""
    return _native.lib().pm_linear_recurrence_workspace_bytes(n_seqs, T, C, packed, x_code)


def _launch(call, xd, gd, cu, s0, slots, n_slots, bad, s_out, n_seqs, T, C, out_dtype, keep, cu_flag=None):
    """The forward on device tensors: ``(h, kept)``; ``s_out`` is written. xd and gd are
    (n_seqs, T, C), or packed (1, T, C) with ``cu``, whose check goes to ``cu_flag``."""
    ptr = _k._ptr
    h = torch.empty_like(xd, dtype=out_dtype, memory_format=torch.contiguous_format)
    spans = -(-T // _native.RECURRENCE_SPAN)
    kept = torch.empty((n_seqs, spans, C), dtype=torch.float32, device=call.device) if keep else None
    xc, gc = _k._code(xd.dtype), _k._code(gd.dtype)
    nbytes = _ws_bytes(n_seqs, T, C, cu is not None, xc)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=call.device) if nbytes else None
    (x_sb, x_st, _), (g_sb, g_st, _) = xd.stride(), gd.stride()
    _native.check(_native.lib().pm_linear_recurrence_varlen(
        xd.data_ptr(), gd.data_ptr(), ptr(cu), ptr(s0), ptr(slots), n_slots, ptr(bad), ptr(cu_flag), h.data_ptr(),
        s_out.data_ptr(), ptr(kept), n_seqs, T, C, x_sb, x_st, g_sb, g_st, xc, gc, _k._code(out_dtype), ptr(ws), nbytes,
        _k._stream(call.device)))
    return h, kept


def _forward(x, g, state, out_dtype, keep=False):
    batch, seq, chan = _check(x, g, state, 3)
    odt = _k._out_dtype(out_dtype)
    call = _k._Call(x, g, state)
    xt, gt = _types(x, g)
    with _k._on(call.device):
        xd, gd, sd = _rows(call, x, xt), _rows(call, g, gt), call.dev(state, torch.float32)
        s_out = torch.empty((batch, chan), dtype=torch.float32, device=call.device)
        h, kept = _launch(call, xd, gd, None, sd, None, 0, None, s_out, batch, seq, chan, odt, keep)
    return call, xd, gd, kept, h, s_out


def _launch_bwd(call, xd, gd, kept, gh, gs, h_dtype):
    """The backward on device tensors: ``(gx, gg, gs0)``."""
    batch, seq, chan = xd.shape
    ptr = _k._ptr
    gx = torch.empty_like(xd, memory_format=torch.contiguous_format)
    gg = torch.empty_like(gd, memory_format=torch.contiguous_format)
    gs0 = torch.empty((batch, chan), dtype=torch.float32, device=call.device)
    xc, gc = _k._code(xd.dtype), _k._code(gd.dtype)
    nbytes = _ws_bytes(batch, seq, chan, False, xc)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=call.device) if nbytes else None
    (x_sb, x_st, _), (g_sb, g_st, _) = xd.stride(), gd.stride()
    _native.check(_native.lib().pm_linear_recurrence_bwd(
        xd.data_ptr(), gd.data_ptr(), ptr(kept), ptr(gh), ptr(gs), gx.data_ptr(), gg.data_ptr(), gs0.data_ptr(), batch,
        seq, chan, x_sb, x_st, g_sb, g_st, xc, gc, _k._code(h_dtype), ptr(ws), nbytes, _k._stream(call.device)))
    return gx, gg, gs0


class _LinearRecurrence(torch.autograd.Function):
    """``linear_recurrence`` as a differentiable op; gradients in each input's type."""

    @staticmethod
    def forward(ctx, x, g, state, out_dtype):
        call, xd, gd, kept, h, s = _forward(x, g, state, out_dtype, keep=True)
        ctx.save_for_backward(xd, gd, kept)
        ctx.saved = (xd.dtype, gd.dtype, xd.shape, kept.shape)
        ctx.call, ctx.h_dtype = call, h.dtype
        ctx.set_materialize_grads(False)  # a missing gradient is None, not a tensor of zeros
        # (the type and device of each input's gradient, where it is not as the backward gives it)
        as_given = xd is x and gd is g and (state is None or (
            isinstance(state, torch.Tensor) and state.dtype == torch.float32 and state.device == call.device))
        ctx.like = None if as_given else [(t.dtype, t.device) if isinstance(t, torch.Tensor) else None
                                          for t in (x, g, state)]
        return call.out(h), call.out(s)

    @staticmethod
    @_k._once
    def backward(ctx, gh, gs):
        call, (xd, gd, kept) = ctx.call, ctx.saved_tensors
        xt, gt, shape, kept_shape = ctx.saved
        gpu = call.device.index
        with _k._on(call.device):
            if not (xd.dtype == xt and xd.shape == shape and xd.get_device() == gpu and gd.dtype == gt
                    and gd.shape == shape and gd.get_device() == gpu and kept.dtype == torch.float32
                    and kept.shape == kept_shape and kept.get_device() == gpu and kept.is_contiguous()
                    and (shape[2] <= 1 or xd.stride(2) == gd.stride(2) == 1)):
                # (saved-tensor hooks may hand back another layout, or copies elsewhere or of another type)
                xd, gd, kept = (_k._as_saved(t, dtype, size, call.device) for t, dtype, size in (
                    (xd, xt, shape), (gd, gt, shape), (kept, torch.float32, kept_shape)))
                xd, gd, kept = _rows(call, xd, xt), _rows(call, gd, gt), kept.contiguous()
            grads = _launch_bwd(call, xd, gd, kept, call.dev(gh), call.dev(gs), ctx.h_dtype)
        if ctx.like is not None:
            grads = [t if like is None else t.to(device=like[1], dtype=like[0]) for t, like in zip(grads, ctx.like)]
        x, g, state, _ = ctx.needs_input_grad
        return grads[0] if x else None, grads[1] if g else None, grads[2] if state else None, None


def linear_recurrence(x, g, state=None, *, out_dtype=None):
    """``h_t = exp(g_t) h_{t-1} + x_t`` over (batch, seq, channels) ``x`` and log-gates ``g``.

    state: (batch, channels) fp32 initial state, zeros if None. Returns ``(h, next_state)``: h
    shaped like x (fp32 unless ``out_dtype`` asks for bf16), next_state (batch, channels) fp32.
    Gates at or below zero keep the state bounded; positive ones are accepted as long as the
    products of a sequence's gates stay finite in fp32. A gate below 2^-126 (g < -87.3) counts as
    closed: it leaves nothing of the state before (NaN of an infinite one). Differentiable: when autograd records
    and a torch input requires grad, the backward is ``linear_recurrence_bwd``.
    """
    if _k._wants_grad(x, g, state):
        return _LinearRecurrence.apply(x, g, state, out_dtype)
    call, _, _, _, h, s = _forward(x, g, state, out_dtype)
    return call.out(h), call.out(s)


def linear_recurrence_fwd(x, g, state=None, *, out_dtype=None):
    """Explicit forward of the VJP pair: ``((h, next_state), residual)`` for
    ``linear_recurrence_bwd``. The residual keeps x, g and one state in every 128 tokens, not h."""
    call, xd, gd, kept, h, s = _forward(x, g, state, out_dtype, keep=True)
    residual = _RecurrenceResidual(call.out(xd), call.out(gd), call.out(kept), h.dtype)
    return (call.out(h), call.out(s)), residual


def linear_recurrence_bwd(residual: _RecurrenceResidual, grads):
    """Backward of the VJP pair: ``grads = (gh, gs)``, dL/dh (batch, seq, channels) and
    dL/dnext_state (batch, channels), either may be None. Returns ``(gx, gg, gstate)``, in x's
    and g's type and fp32. With d_t = gh_t + exp(g_{t+1}) d_{t+1}: gx_t = d_t and
    gg_t = d_t exp(g_t) h_{t-1}, h recomputed in fp32 from the kept states."""
    gh, gs = grads
    x, g, kept = residual.x, residual.g, residual.kept
    batch, seq, chan = _check(x, g, None, 3)
    spans = -(-seq // _native.RECURRENCE_SPAN)
    if _k._shape(kept) != (batch, spans, chan):
        raise _k.KernelError(f"kept states {_k._shape(kept)} != {(batch, spans, chan)}")
    if gh is not None and _k._shape(gh) != (batch, seq, chan):
        raise _k.KernelError(f"grad of output shape {_k._shape(gh)} != {(batch, seq, chan)}")
    if gs is not None and _k._shape(gs) != (batch, chan):
        raise _k.KernelError(f"grad of state shape {_k._shape(gs)} != {(batch, chan)}")
    call = _k._Call(x, g, kept, gh, gs)
    xt, gt = _types(x, g)
    with _k._on(call.device):
        grads = _launch_bwd(call, _rows(call, x, xt), _rows(call, g, gt), call.dev(kept, torch.float32),
                            call.dev(gh, residual.h_dtype), call.dev(gs, torch.float32), residual.h_dtype)
    return tuple(call.out(t) for t in grads)


def _packed(x, g, cu_seqlens):
    """Shapes of a packed call and its offsets as ``(n_tok, chan, n_seqs, offsets)``: the host's
    checked here, a GPU tensor given back for the device's check."""
    xs = _k._shape(x)
    if _k._shape(g) != xs or len(xs) not in (2, 3) or (len(xs) == 3 and xs[0] != 1):
        raise _k.KernelError(f"packed x and g must both be (N, C) or (1, N, C); got {xs} and {_k._shape(g)}")
    n_tok, chan = xs[-2:]
    if n_tok >= 2**31:
        raise _k.KernelError("cu_seqlens exceeds int32")
    if isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.device.type == "cuda":
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
            raise _k.KernelError("cu_seqlens must be a 1-D array of n_seqs + 1 offsets")
        if cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise _k.KernelError(f"cu_seqlens must be an integer array, got {cu_seqlens.dtype}")
        return n_tok, chan, cu_seqlens.numel() - 1, cu_seqlens
    host = cu_seqlens.detach().numpy() if isinstance(cu_seqlens, torch.Tensor) else np.asarray(cu_seqlens)
    if not np.issubdtype(host.dtype, np.integer):
        raise _k.KernelError(f"cu_seqlens must be an integer array, got {host.dtype}")
    host = host.astype(np.int64)
    _k._validate_cu(host, n_tok)
    return n_tok, chan, host.size - 1, host


def _offsets(call, cu, n_seqs, n_tok, chan):
    """int32 offsets on the device and, for those of a GPU tensor, the flag of ``check_varlen`` that
    the launch is to set (a call that launches nothing is checked here)."""
    if isinstance(cu, np.ndarray):
        return torch.from_numpy(cu.astype(np.int32)).to(call.device), None
    cu, flag = _k._offsets_i32(cu, n_tok), _k._varlen_flag(call.device)
    if n_seqs == 0 or chan == 0:
        _native.check(_native.lib().pm_varlen_check(cu.data_ptr(), n_seqs, n_tok, flag.data_ptr(),
                                                    _k._stream(call.device)))
        return cu, None
    return cu, flag


def linear_recurrence_varlen(x, g, cu_seqlens, state=None, *, out_dtype=None):
    """Packed batch of independent sequences, the state starting anew at every boundary.

    x, g: (N, C) or (1, N, C); cu_seqlens and its checks as ``chunked_delta_rule_varlen``;
    state: None (zeros) or (n_seqs, C). Returns ``(h, final_states)``, h shaped like x and
    final_states (n_seqs, C) fp32 (an empty sequence's is its initial state). Forward only:
    inputs that require grad are refused while autograd records.
    """
    if _k._wants_grad(x, g, state):
        raise _k.KernelError("linear_recurrence_varlen is forward only: call it under torch.no_grad()")
    n_tok, chan, n_seqs, cu = _packed(x, g, cu_seqlens)
    if state is not None and _k._shape(state) != (n_seqs, chan):
        raise _k.KernelError(f"state shape {_k._shape(state)} != {(n_seqs, chan)}")
    odt = _k._out_dtype(out_dtype)
    call = _k._Call(x, g, state, cu_seqlens)
    xt, gt = _types(x, g)
    with _k._on(call.device):
        xd, gd = (t if t.dim() == 3 else t[None] for t in (_rows(call, x, xt), _rows(call, g, gt)))
        sd = call.dev(state, torch.float32)
        s_out = torch.empty((n_seqs, chan), dtype=torch.float32, device=call.device)
        cu, flag = _offsets(call, cu, n_seqs, n_tok, chan)
        h, _ = _launch(call, xd, gd, cu, sd, None, 0, None, s_out, n_seqs, n_tok, chan, odt, False, flag)
    return call.out(h.reshape(_k._shape(x))), call.out(s_out)


def linear_recurrence_step(x, g, state, *, out_dtype=None):
    """One token: ``state = exp(g) state + x`` for (B, C) ``x`` and ``g``, ``state`` (B, C) fp32
    updated in place as in ``delta_rule_step``; returns h (B, C), the new state in fp32 or
    ``out_dtype``. Forward only, as ``linear_recurrence_varlen``."""
    if _k._wants_grad(x, g, state):
        raise _k.KernelError("linear_recurrence_step is forward only: call it under torch.no_grad()")
    batch, chan = _check(x, g, state, 2)
    if state is None:
        raise _k.KernelError(f"state shape None != {(batch, chan)}")
    in_place = isinstance(state, torch.Tensor) and state.device.type == "cuda"
    if in_place and (state.dtype != torch.float32 or not state.is_contiguous()):
        raise _k.KernelError("state must be a contiguous fp32 tensor to be updated in place")
    if isinstance(state, np.ndarray) and state.dtype != np.float32:
        raise _k.KernelError("state must be fp32 to be updated in place")
    odt = _k._out_dtype(out_dtype)
    call = _k._Call(x, g, state)
    xt, gt = _types(x, g)
    with _k._on(call.device):
        xd, gd = _rows(call, x, xt), _rows(call, g, gt)
        sd = state if in_place else call.dev(state, torch.float32)
        h = torch.empty((batch, chan), dtype=odt, device=call.device)
        _step(_k._ptr(sd), None, 0, xd, gd, h, _k._stream(call.device))
        if not in_place:
            host = sd.cpu()
            if isinstance(state, np.ndarray):
                state[...] = host.numpy()
            else:
                state.copy_(host)
    return call.out(h)


def _step(state: int | None, slots, n_slots, xd, gd, h, stream):
    """One token on device tensors; ``state`` is the states' address."""
    batch, chan = xd.shape
    _native.check(_native.lib().pm_linear_recurrence_step(
        state, _k._ptr(slots), n_slots, xd.data_ptr(), gd.data_ptr(), h.data_ptr(), batch, chan, xd.stride(0), gd.stride(0),
        _k._code(xd.dtype), _k._code(gd.dtype), _k._code(h.dtype), stream))
