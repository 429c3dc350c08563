"""Serving-side state cache of the linear-attention layers on MI355X.

The reference's serving spec (``spec/13-serving.md`` item 4) and its SGLang
fork (``sglang-fork/sglang_fork/model_def.py``, layer kinds only) describe
the consumer of the decode step: every linear-attention layer keeps one
fixed-size state per request (``(H, D, D)`` fp32, as ``kernels/__init__.py``
carries it), so a serving engine holds those states in a pool and decodes a
batch of requests through a slot table, and parks idle sessions' states in
host memory. ``LinearStateCache`` is that pool on one GPU:

* ``pool``: ``(n_layers, n_slots, H, D, D)`` fp32 in HBM (64 KiB per slot and
  layer at H = 1, D = 128);
* ``alloc`` / ``free`` / ``reset``: slot bookkeeping on the host;
* ``prefill``: runs a prompt through the forward (the chunked MFMA kernel for
  bf16 with D in {64, 128}), starting from and ending in the requests' slots;
  with the slots and ``cu_seqlens`` as GPU tensors it never synchronises with
  the host, so it can be captured in a HIP graph (an out-of-range device slot
  computes from a zero state into a spare slot past the pool's end, leaves the
  pool untouched, and is reported by ``check_slots``);
* ``decode``: one token per request, in place, through ``pm_delta_step_slots``
  (allocation-free with ``out=``, no host synchronisation, so it can be
  captured in a HIP graph with a fixed slot tensor whose contents change
  between replays; slots outside ``[0, n_slots)`` are padding);
* ``swap_out`` / ``swap_in``: park states in pinned host memory and restore
  them (the spec's tier-2 parking of long sessions).

``RecurrenceStateCache`` is the same for layers of ``kernels.linear_recurrence``, whose state is
a vector of C channels (``(n_layers, n_slots, C)`` fp32): its ``prefill`` reads and writes the
slots in the kernel, without gathering them first.
"""

from __future__ import annotations

import heapq

import torch

from prometheus_amd import _native, kernels
from prometheus_amd.kernels import recurrence

__all__ = ["LinearStateCache", "RecurrenceStateCache"]


class _SlotPool:
    """Slots of per-request states, each ``state`` fp32 per layer: bookkeeping and tiering."""

    def __init__(self, n_layers: int, n_slots: int, state: tuple, device):
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.n_layers, self.n_slots, self._state = n_layers, n_slots, state
        # one spare slot past the end: out-of-range device slot indices land there
        self._pool = torch.zeros((n_layers, n_slots + 1, *state), dtype=torch.float32, device=device)
        self.pool = self._pool[:, :n_slots]
        self._gpu = self._pool.get_device()  # (-1 on the host)
        self._bad_slot = torch.zeros(1, dtype=torch.int32, device=device)
        # a min-heap: alloc hands out the lowest free slots, so that a batch admitted in
        # order decodes through an increasing slot table, which walks the pool in address
        # order (at cfg4, 0.71 of HBM against 0.69 for a random table)
        self._free = list(range(n_slots))
        self._used: set[int] = set()

    # ---- bookkeeping ----
    @property
    def n_free(self) -> int:
        return len(self._free)

    def alloc(self, n: int = 1) -> list[int]:
        """Take ``n`` free slots; their states are zero (a fresh request)."""
        if n < 0 or n > len(self._free):
            raise RuntimeError(f"cannot allocate {n} slots ({len(self._free)} free)")
        got = [heapq.heappop(self._free) for _ in range(n)]
        self._used.update(got)
        if got:
            self.reset(got)
        return got

    def free(self, slots) -> None:
        for s in self._ids(slots):
            if s not in self._used:
                raise ValueError(f"slot {s} is not allocated")
            self._used.remove(s)
            heapq.heappush(self._free, s)

    def reset(self, slots) -> None:
        idx = self._index(slots)
        self._pool[:, idx] = 0.0

    def check_slots(self) -> None:
        """Raise ``ValueError`` if a GPU slot tensor given to ``prefill`` or ``reset`` since
        the last check held an index outside ``[0, n_slots)`` (synchronises; clears)."""
        if int(self._bad_slot.item()):
            self._bad_slot.zero_()
            raise ValueError(f"a device slot index was outside [0, {self.n_slots})")

    # ---- tiering ----
    def swap_out(self, slots) -> torch.Tensor:
        """The slots' states of every layer, copied to pinned host memory:
        ``(n_layers, n, *state)``. The slots stay allocated."""
        idx = self._index(slots)
        host = torch.empty((self.n_layers, len(idx), *self._state), dtype=torch.float32, pin_memory=True)
        host.copy_(self._pool[:, idx])
        return host

    def swap_in(self, slots, saved: torch.Tensor) -> None:
        idx = self._index(slots)
        want = (self.n_layers, len(idx), *self._state)
        if tuple(saved.shape) != want:
            raise ValueError(f"saved states {tuple(saved.shape)} != {want}")
        self._pool[:, idx] = saved.to(self._pool.device, dtype=torch.float32)

    # ---- helpers ----
    def _ids(self, slots) -> list[int]:
        ids = [int(s) for s in (slots.tolist() if isinstance(slots, torch.Tensor) else slots)]
        for s in ids:
            if not 0 <= s < self.n_slots:
                raise ValueError(f"slot {s} outside [0, {self.n_slots})")
        return ids

    def _index(self, slots) -> torch.Tensor:
        if isinstance(slots, torch.Tensor) and slots.device.type == "cuda":
            # checked on the device: an index outside [0, n_slots) becomes the spare slot
            if slots.dim() != 1 or slots.dtype not in (torch.int32, torch.int64):
                raise ValueError("a GPU slot tensor must be 1-D int32 or int64")
            if slots.device != self._pool.device:
                raise ValueError("slots must be on the pool's device")
            idx = slots.long()
            bad = (idx < 0) | (idx >= self.n_slots)
            self._bad_slot.bitwise_or_(bad.any().to(torch.int32))
            return torch.where(bad, torch.full_like(idx, self.n_slots), idx)
        return torch.tensor(self._ids(slots), dtype=torch.long, device=self._pool.device)

    def _check_layer(self, layer: int) -> None:
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} outside [0, {self.n_layers})")

    def _check_cuda(self, *xs) -> None:
        gpu = self._gpu
        if gpu < 0:
            raise RuntimeError("the state cache computes on a HIP GPU; this pool is on the host")
        for x in xs:
            if not (isinstance(x, torch.Tensor) and x.get_device() == gpu):
                raise ValueError("inputs must be tensors on the pool's device")


class LinearStateCache(_SlotPool):
    """Per-request recurrent states of ``n_layers`` linear-attention layers."""

    def __init__(self, n_layers: int, n_slots: int, heads: int, dim: int, device=None):
        if n_layers < 1 or n_slots < 1 or heads < 1 or dim < 1:
            raise ValueError("n_layers, n_slots, heads and dim must be >= 1")
        super().__init__(n_layers, n_slots, (heads, dim, dim), device)
        self.heads, self.dim = heads, dim

    def prefill(self, layer: int, slots, q, k, v, beta, cu_seqlens=None, config=None):
        """Run prompts through the forward from the slots' states into them.

        Fixed length: q, k, v ``(n, T, H, D)``, beta ``(n, T, H)``, one request per
        row. Packed: q, k, v ``(1, N, H, D)`` with ``cu_seqlens`` ``(n + 1,)``.
        Returns the output ``(.., H, D)`` fp32. ``slots`` may be a list of ints or a
        GPU int tensor; with GPU ``slots`` and ``cu_seqlens`` nothing here waits for
        the device (see ``check_slots`` and ``kernels.check_varlen``).
        """
        self._check_layer(layer)
        idx = self._index(slots)
        self._check_cuda(q, k, v, beta)
        self._pool[layer, self.n_slots].zero_()  # the spare slot: a fresh state
        s0 = self._pool[layer, idx]  # gathered copy (n, H, D, D)
        if cu_seqlens is None:
            o, s = kernels.chunked_delta_rule(q, k, v, beta, s0, config)
        else:
            o, s = kernels.chunked_delta_rule_varlen(q, k, v, beta, cu_seqlens, s0, config)
        self._pool[layer, idx] = s
        return o

    def decode(self, layer: int, slots: torch.Tensor, q, k, v, beta, out=None):
        """One token per request: q, k, v ``(B, H, D)``, beta ``(B, H)``, ``slots``
        an int32 GPU tensor ``(B,)``. Updates the states in place and returns
        ``out`` ``(B, H, D)`` fp32 (allocated when None)."""
        self._check_layer(layer)
        self._check_cuda(q, k, v, beta, slots)
        b = slots.shape[0] if slots.dim() == 1 else -1
        if b < 0 or slots.dtype != torch.int32 or not slots.is_contiguous():
            raise ValueError("slots must be a contiguous int32 tensor of shape (B,)")
        want = (b, self.heads, self.dim)
        for name, x in (("q", q), ("k", k), ("v", v)):
            if tuple(x.shape) != want or not x.is_contiguous():
                raise ValueError(f"{name} must be contiguous {want}, got {tuple(x.shape)}")
        if q.dtype != k.dtype or q.dtype != v.dtype or q.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("q, k, v must share one dtype, fp32 or bf16")
        if tuple(beta.shape) != (b, self.heads) or beta.dtype != torch.float32 or not beta.is_contiguous():
            raise ValueError(f"beta must be contiguous fp32 {(b, self.heads)}")
        if out is None:
            out = torch.empty(want, dtype=torch.float32, device=q.device)
        elif tuple(out.shape) != want or out.dtype != torch.float32 or not out.is_contiguous():
            raise ValueError(f"out must be contiguous fp32 {want}")
        with kernels._on(q.device):
            rc = _native.lib().pm_delta_step_slots(
                self.pool[layer].data_ptr(), slots.data_ptr(), self.n_slots, q.data_ptr(), k.data_ptr(),
                v.data_ptr(), beta.data_ptr(), out.data_ptr(), b, self.heads, self.dim,
                _native.DTYPE_BF16 if q.dtype == torch.bfloat16 else _native.DTYPE_F32,
                kernels._stream(q.device),
            )
        _native.check(rc)
        return out


class RecurrenceStateCache(_SlotPool):
    """Per-request states of ``n_layers`` layers of the elementwise linear recurrence."""

    def __init__(self, n_layers: int, n_slots: int, channels: int, device=None):
        if n_layers < 1 or n_slots < 1 or channels < 1:
            raise ValueError("n_layers, n_slots and channels must be >= 1")
        super().__init__(n_layers, n_slots, (channels,), device)
        self.channels = channels

    def prefill(self, layer: int, slots, x, g, cu_seqlens=None, *, out_dtype=None):
        """Run prompts through the recurrence from the slots' states into them, in place.

        Fixed length: x, g ``(n, T, C)``, one request per row. Packed: ``(N, C)`` or ``(1, N, C)``
        with ``cu_seqlens`` ``(n + 1,)``. Returns h shaped like x. ``slots`` (each at most once)
        may be a list of ints or a GPU int tensor; with GPU ``slots`` and ``cu_seqlens`` nothing
        here waits for the device: a request whose slot is out of range starts from a zero state,
        leaves the pool untouched and is reported by ``check_slots``.
        """
        self._check_layer(layer)
        odt = kernels._out_dtype(out_dtype)
        if isinstance(slots, torch.Tensor) and slots.device.type == "cuda":
            if slots.dim() != 1 or slots.dtype not in (torch.int32, torch.int64):
                raise ValueError("a GPU slot tensor must be 1-D int32 or int64")
            n = slots.shape[0]
        else:
            slots = self._ids(slots)
            n = len(slots)
            if len(set(slots)) != n:
                raise ValueError("a slot may be given once")
        if kernels._wants_grad(x, g):
            raise ValueError("prefill is forward only: call it under torch.no_grad()")
        if cu_seqlens is None:
            _, seq, chan = recurrence._check(x, g, None, 3)
            n_seqs, cu = x.shape[0], None
        else:
            seq, chan, n_seqs, cu = recurrence._packed(x, g, cu_seqlens)
        if chan != self.channels:
            raise ValueError(f"x has {chan} channels, the cache {self.channels}")
        if n_seqs != n:
            raise ValueError(f"{n} slots for {n_seqs} prompts")
        self._check_cuda(x, g)
        call = kernels._Call(x, g, cu_seqlens)
        xt, gt = recurrence._types(x, g)
        with torch.cuda.device(call.device):
            if isinstance(slots, list):
                slots = torch.tensor(slots, dtype=torch.int32, device=call.device)
            elif slots.device != self._pool.device:
                raise ValueError("slots must be on the pool's device")
            elif slots.dtype == torch.int64:
                # (clamped: an index past int32 must not come back into range)
                slots = slots.clamp(-1, self.n_slots).to(torch.int32)
            xd, gd = (t if t.dim() == 3 else t[None] for t in (recurrence._rows(call, x, xt),
                                                               recurrence._rows(call, g, gt)))
            flag = None
            if cu is not None:
                cu, flag = recurrence._offsets(call, cu, n_seqs, seq, chan)
            pool = self._pool[layer]
            h, _ = recurrence._launch(call, xd, gd, cu, pool, slots.contiguous(), self.n_slots, self._bad_slot, pool,
                                      n_seqs, seq, chan, odt, False, flag)
        return h.reshape(x.shape)

    def decode(self, layer: int, slots: torch.Tensor, x, g, out=None, *, out_dtype=None):
        """One token per request: x, g ``(B, C)``, ``slots`` an int32 GPU tensor ``(B,)``. Updates
        the states in place and returns ``out`` ``(B, C)`` (allocated when None: fp32, or
        ``out_dtype``). Slots outside ``[0, n_slots)`` are padding: no state is touched and their
        rows are zero. Allocation-free with ``out=`` and x and g in a type the kernel takes."""
        self._check_layer(layer)
        if kernels._wants_grad(x, g):
            raise ValueError("decode is forward only: call it under torch.no_grad()")
        self._check_cuda(x, g, slots)
        if slots.dim() != 1 or slots.dtype != torch.int32 or not slots.is_contiguous():
            raise ValueError("slots must be a contiguous int32 tensor of shape (B,)")
        want = (slots.shape[0], self.channels)
        if x.shape != want or g.shape != want:
            raise ValueError(f"x and g must be {want}, got {tuple(x.shape)} and {tuple(g.shape)}")
        if x.dtype not in (torch.float32, torch.bfloat16) or g.dtype not in (torch.float32, x.dtype):
            raise ValueError("x must be fp32 or bf16, and g fp32 or x's type")
        if want[1] > 1 and (x.stride(1) != 1 or g.stride(1) != 1):
            raise ValueError("x and g must have contiguous channels")
        if out is None:
            out = torch.empty_like(x, dtype=kernels._out_dtype(out_dtype), memory_format=torch.contiguous_format)
        elif (tuple(out.shape) != want or out.dtype not in (torch.float32, torch.bfloat16)
              or not out.is_contiguous() or out.device != x.device):
            raise ValueError(f"out must be contiguous fp32 or bf16 {want} on the pool's device")
        with kernels._on(x.device):
            recurrence._step(self._pool.data_ptr() + layer * self._pool.stride(0) * 4, slots, self.n_slots, x, g, out,
                             kernels._stream(x.device))
        return out
