"""GPU tests of the operators beside the delta rule where their kernels change course: tokens around
the tiles' and groups' edges, more tiles than workgroups, many packed sequences, heads in groups,
strides past 32 bits, and both directions in a graph.

Tolerances are the oracle's error bounds for fp32 arithmetic plus half a step of the output's type.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import layer_oracle as ref
from prometheus_amd import kernels

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _host(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _near(got, want, bound, name):
    half = torch.finfo(got.dtype).eps / 2
    g = _host(got)
    off, tol = np.abs(g - want), bound * (1 + half) + half * np.abs(want) + 1e-30
    assert np.isfinite(g).all(), name
    worst = np.unravel_index(np.argmax(off / tol), off.shape) if off.size else None
    assert worst is None or off[worst] <= tol[worst], (name, worst, g[worst], want[worst], off[worst] / tol[worst])


def _inputs(shape, dtype, seed, rate):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g = -rate * torch.rand(shape, generator=gen, device="cuda") ** 3
    return torch.randn(shape, generator=gen, device="cuda").to(dtype), g.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [127, 128, 129, 256, 257, 511, 512, 513, 1025, 8191, 8192, 8193, 8705])
def test_recurrence_around_the_edges_of_tiles_and_groups(T, dtype):
    B, C = 2, 9
    x, g = _inputs((B, T, C), dtype, T, 3e-3)
    s0 = torch.randn(B, C, device="cuda")
    hx, hg, hs = _host(x), _host(g), _host(s0)
    (h, s), res = kernels.linear_recurrence_fwd(x, g, s0, out_dtype=dtype)
    want, _ = ref.recurrence(hx, hg, hs)
    bound = ref.recurrence_bound(hx, hg, hs)
    _near(h, want, bound, "h")
    _near(s, want[:, -1], bound[:, -1], "state")
    gh, gs = torch.randn(B, T, C, device="cuda").to(dtype), torch.randn(B, C, device="cuda")
    got = kernels.linear_recurrence_bwd(res, (gh, gs))
    for name, u, v, w in zip(("gx", "gg", "gs0"), got, ref.recurrence_bwd(hx, hg, hs, _host(gh), _host(gs)),
                             ref.recurrence_bwd_bound(hx, hg, hs, _host(gh), _host(gs))):
        _near(u, v, w, name)
    cu = np.array([0, T // 3, T // 3, T])  # the same tokens packed
    hp, sp = kernels.linear_recurrence_varlen(x[0], g[0], cu, out_dtype=dtype)
    for i in (0, 2):
        a = (hx[:1, cu[i]:cu[i + 1]], hg[:1, cu[i]:cu[i + 1]])
        _near(hp[cu[i]:cu[i + 1]][None], ref.recurrence(*a)[0], ref.recurrence_bound(*a), ("packed", i))
        _near(sp[i:i + 1], ref.recurrence(*a)[1], ref.recurrence_bound(*a)[:, -1], ("packed state", i))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,C", [(2, 3001, 4100), (40, 100, 3000), (20, 200, 3000), (1, 20000, 520)])
def test_recurrence_of_many_tiles_is_that_of_each_channel(B, T, C, dtype):
    """The order of products does not depend on how many tiles run at a time: the same bits."""
    x, g = _inputs((B, T, C), dtype, C, 1e-2)
    s0 = torch.randn(B, C, device="cuda")
    gh, gs = torch.randn(B, T, C, device="cuda").to(dtype), torch.randn(B, C, device="cuda")
    (h, s), res = kernels.linear_recurrence_fwd(x, g, s0, out_dtype=dtype)
    grads = kernels.linear_recurrence_bwd(res, (gh, gs))
    cu = torch.arange(0, B * T + 1, T, dtype=torch.int32, device="cuda")
    hp, sp = kernels.linear_recurrence_varlen(x.flatten(0, 1), g.flatten(0, 1), cu, s0, out_dtype=dtype)
    for b, c in ((0, slice(0, 64)), (B - 1, slice(C - 70, C)), (B // 2, slice(C // 2, C // 2 + 5))):
        part = [t[b:b + 1, ..., c] for t in (x, g, s0)]
        (hb, sb), rb = kernels.linear_recurrence_fwd(*part, out_dtype=dtype)
        assert torch.equal(hb, h[b:b + 1, :, c]) and torch.equal(sb, s[b:b + 1, c])
        for u, v in zip(kernels.linear_recurrence_bwd(rb, (gh[b:b + 1, :, c], gs[b:b + 1, c])), grads):
            assert torch.equal(u, v[b:b + 1, ..., c])
        hq, sq = kernels.linear_recurrence_varlen(x.flatten(0, 1)[:, c], g.flatten(0, 1)[:, c], cu, s0[:, c], out_dtype=dtype)
        assert torch.equal(hq, hp[:, c]) and torch.equal(sq, sp[:, c])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_packed_more_sequences_than_threads(dtype):
    rng = np.random.default_rng(1)
    n, C = 1300, 12
    lens = rng.integers(0, 5, n)
    lens[[7, 600, 1299]] = 700, 513, 90
    cu = np.concatenate([[0], np.cumsum(lens)])
    x, g = _inputs((int(cu[-1]), C), dtype, 3, 0.2)
    s0 = torch.randn(n, C, device="cuda")
    h, s = kernels.linear_recurrence_varlen(x, g, cu, s0, out_dtype=dtype)
    hx, hg, hs = _host(x), _host(g), _host(s0)
    want, bound = np.zeros_like(hx), np.zeros_like(hx)
    end, off = hs.copy(), np.zeros_like(hs)
    for i in range(n):
        a, z = cu[i], cu[i + 1]
        if a < z:
            args = hx[None, a:z], hg[None, a:z], hs[i:i + 1]
            want[a:z], bound[a:z] = ref.recurrence(*args)[0][0], ref.recurrence_bound(*args)[0]
            end[i], off[i] = want[z - 1], bound[z - 1]
    _near(h, want, bound, "h")
    _near(s, end, off, "state")


def test_recurrence_strides_past_32_bits():
    B, T, C = 2, 300, 8
    buf = torch.empty(2**31 + 300 * 2**23, dtype=BF16, device="cuda")
    for shape in ((2**31, C, 1), (2**23 * 5, 2**23, 1)):
        x, g = buf.as_strided((B, T, C), shape), buf.as_strided((B, T, C), shape, 2**22)
        vx, vg = _inputs((B, T, C), BF16, 1, 0.1)
        x.copy_(vx), g.copy_(vg)
        gh = torch.randn(B, T, C, device="cuda")
        want, res = kernels.linear_recurrence_fwd(x.contiguous(), g.contiguous())
        got, res2 = kernels.linear_recurrence_fwd(x, g)
        assert all(torch.equal(u, v) for u, v in zip(got, want))
        for u, v in zip(kernels.linear_recurrence_bwd(res2, (gh, None)), kernels.linear_recurrence_bwd(res, (gh, None))):
            assert torch.equal(u, v)


def test_both_directions_replayed_from_a_graph():
    B, T, C, H, D = 2, 9000, 200, 4, 64
    x, g = _inputs((B, T, C), BF16, 2, 1e-2)
    gh = torch.randn(B, T, C, device="cuda").to(BF16)
    q = torch.randn(B, 700, H, D, device="cuda").to(BF16)
    w, table = torch.ones(D, device="cuda"), kernels.rotation_table(700, D)

    def work():
        (h, s), res = kernels.linear_recurrence_fwd(x, g, out_dtype=BF16)
        outs, heads = kernels.norm_rotate_fwd(q, q, table, norm="rms", q_weight=w)
        return (h, s, *kernels.linear_recurrence_bwd(res, (gh, s)), *outs, *kernels.norm_rotate_bwd(heads, outs)[:3])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for _ in range(4):
        x.copy_(torch.randn(B, T, C, device="cuda"))
        q.copy_(torch.randn(B, 700, H, D, device="cuda"))
        want = work()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(outs, want))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,Hq,Hk,D,R,interleaved", [
    (2, 4100, 16, 4, 128, 128, False), (1, 2100, 7, 8, 256, 64, True), (3, 1500, 11, 12, 80, 40, False),
    (1, 9000, 8, 8, 33, 32, False), (2, 4500, 8, 4, 96, 0, False), (1, 30000, 4, 4, 16, 16, True)])
def test_heads_in_groups(B, T, Hq, Hk, D, R, interleaved, dtype):
    gen = torch.Generator(device="cuda").manual_seed(D)
    q, k = (torch.randn(B, T, H, D, generator=gen, device="cuda").to(dtype) for H in (Hq, Hk))
    wq = 1 + 0.2 * torch.randn(D, generator=gen, device="cuda")
    wk = 1 + 0.2 * torch.randn(D, generator=gen, device="cuda")
    table = kernels.rotation_table(T, R) if R else None
    opts = dict(norm="rms", q_weight=wq, k_weight=wk, interleaved=interleaved)
    outs, res = kernels.norm_rotate_fwd(q, k, table, **opts)
    gz = [torch.randn(x.shape, generator=gen, device="cuda").to(dtype) for x in (q, k)]
    grads = kernels.norm_rotate_bwd(res, gz)
    assert all(torch.equal(u, v) for u, v in zip(grads, kernels.norm_rotate_bwd(res, gz)))
    # a call of few rows takes its heads one by one: rows alike
    few = kernels.norm_rotate(q[:, :3], k[:, :3], table, **opts)
    assert all(torch.equal(u[:, :3], v) for u, v in zip(outs, few))
    # the oracle on some tokens (positions named), and on all for the weights' sums
    at = np.unique(np.linspace(0, T - 1, 40).astype(int))
    pos = None if table is None else np.broadcast_to(at, (B, at.size))
    for i, (x, w) in enumerate(((q, wq), (k, wk))):
        rest = (_host(table), pos, "rms", _host(w), 1e-6, interleaved)
        hx, hz = _host(x[:, at]), _host(gz[i][:, at])
        _near(outs[i][:, at], ref.head_norm(hx, *rest), ref.head_norm_bound(hx, *rest), "qk"[i])
        _near(grads[i][:, at], ref.head_norm_bwd(hx, hz, *rest)[0], ref.head_norm_bwd_bound(hx, hz, *rest)[0], ("gq", "gk")[i])
    full = (_host(k), _host(gz[1]), _host(table), np.broadcast_to(np.arange(T), (B, T)), "rms", _host(wk), 1e-6, interleaved)
    _near(grads[3], ref.head_norm_bwd(*full)[1], ref.head_norm_bwd_bound(*full)[1], "gwk")


def test_heads_strides_past_32_bits():
    B, T, H, D = 2, 5, 3, 64
    buf = torch.empty(2**31 + 2**20, dtype=BF16, device="cuda")
    table = kernels.rotation_table(T, D)
    for strides in ((2**31, H * D, D, 1), (D, 2**28, 2**29 + 64, 1)):
        q = buf.as_strided((B, T, H, D), strides)
        q.copy_(torch.randn(B, T, H, D, device="cuda"))
        want, res = kernels.norm_rotate_fwd(q.contiguous(), q.contiguous(), table)
        got, res2 = kernels.norm_rotate_fwd(q, q, table)
        assert all(torch.equal(u, v) for u, v in zip(got, want))
        for u, v in zip(kernels.norm_rotate_bwd(res2, got)[:2], kernels.norm_rotate_bwd(res, got)[:2]):
            assert torch.equal(u, v)


@pytest.mark.parametrize("N,C", [(400, 16), (3000, 8), (0, 8), (400, 0)])
def test_malformed_device_offsets_are_named(N, C):
    x = torch.randn(N, C, device="cuda")
    kernels.check_varlen()
    for cu, what in (([1, N], r"cu_seqlens\[0\]"), ([0, N + 1], r"cu_seqlens\[-1\].*outside"), ([0, N + 7, N], "outside"),
                     ([0, 2, 1, N], "decreasing"), ([-1, N], r"cu_seqlens\[0\].*outside"), ([N + 1], r"cu_seqlens\[0\]"),
                     ([0, N, N - 1], r"cu_seqlens\[-1\].*decreasing")):
        kernels.linear_recurrence_varlen(x, -x.abs(), torch.tensor(cu, dtype=torch.int32, device="cuda"))
        with pytest.raises(kernels.KernelError, match=what):
            kernels.check_varlen()
    for cu in ([0, N], [0, 0, N, N]):
        kernels.linear_recurrence_varlen(x, -x.abs(), torch.tensor(cu, device="cuda"))
        kernels.check_varlen()


def test_gradients_of_gradients_are_refused():
    x = torch.randn(1, 9, 4, device="cuda", requires_grad=True)
    h, _ = kernels.linear_recurrence(x, -x.abs())
    (gx,) = torch.autograd.grad(h.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate twice"):
        gx.sum().backward()
    q = torch.randn(1, 5, 2, 8, device="cuda", requires_grad=True)
    zq, _ = kernels.norm_rotate(q, q)
    (gq,) = torch.autograd.grad(zq.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate twice"):
        gq.sum().backward()


@pytest.mark.parametrize("where", ["input", "gate", "state"])
def test_gradients_come_in_each_input_s_type_and_place(where):
    """Inputs on the host, of another type or not contiguous, and tensors that hooks pack."""
    base = {"input": torch.randn(2, 300, 7), "gate": -torch.rand(2, 300, 7), "state": torch.randn(2, 7)}
    want = [t.cuda().requires_grad_(True) for t in base.values()]
    h, s = kernels.linear_recurrence(*want)
    grads = torch.autograd.grad(h.square().sum() + s.sum(), want)
    for change in (lambda t: t.double(), lambda t: t.cpu(), lambda t: t.transpose(0, -1).contiguous().transpose(0, -1)):
        args = [change(t.cuda()) if n == where else t.cuda() for n, t in base.items()]
        args = [t.detach().requires_grad_(True) for t in args]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
            h, s = kernels.linear_recurrence(*args)
        got = torch.autograd.grad(h.square().sum() + s.sum(), args)
        for g, a, w in zip(got, args, grads):
            assert g.dtype == a.dtype and g.device == a.device
            assert torch.equal(g.cuda().float(), w)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_packed_sequences_do_not_reach_each_other(dtype):
    """NaN and infinities of a sequence, in its state, tokens or gates, leave the others' bits alone."""
    lens = [3, 509, 1, 4, 700, 8, 2, 100, 1500, 37]
    cu = np.concatenate([[0], np.cumsum(lens)])
    C, n = 72, len(lens)
    x, g = _inputs((int(cu[-1]), C), dtype, 11, 0.05)
    s0 = torch.randn(n, C, device="cuda")
    want, end = kernels.linear_recurrence_varlen(x, g, cu, s0, out_dtype=dtype)
    for i, value in ((0, torch.nan), (1, torch.inf), (4, -torch.inf), (7, torch.nan), (8, torch.inf)):
        y, gate, s = x.clone(), g.clone(), s0.clone()
        y[cu[i]:cu[i + 1], ::3] = value
        gate[cu[i]:cu[i + 1], 1::3] = value
        s[i, 2::3] = value
        h, last = kernels.linear_recurrence_varlen(y, gate, cu, s, out_dtype=dtype)
        others = torch.ones(int(cu[-1]), dtype=torch.bool, device="cuda")
        others[cu[i]:cu[i + 1]] = False
        assert torch.equal(h[others], want[others])
        keep = torch.arange(n, device="cuda") != i
        assert torch.equal(last[keep], end[keep])
        assert not torch.isfinite(h[cu[i]:cu[i + 1], ::3]).any() and not torch.isfinite(last[i, ::3]).any()


@pytest.mark.parametrize("T", [100, 900, 9000])
def test_backward_again_and_in_a_graph(T):
    """A second backward of the same graph, and one that a captured graph replays, set up their own."""
    x, g = _inputs((2, T, 136), BF16, T, 1e-2)
    x, g = x.requires_grad_(True), g.requires_grad_(True)
    gh = torch.randn(2, T, 136, device="cuda").to(BF16)
    _, res = kernels.linear_recurrence_fwd(x.detach(), g.detach(), out_dtype=BF16)
    want = kernels.linear_recurrence_bwd(res, (gh, None))[:2]

    def check(got, want):
        assert all(torch.equal(u, v) for u, v in zip(got, want))

    h, _ = kernels.linear_recurrence(x, g, out_dtype=BF16)
    for _ in range(3):
        check(torch.autograd.grad(h, (x, g), gh, retain_graph=True), want)
    with pytest.raises(RuntimeError, match="second time|already been freed"):
        torch.autograd.grad(h, (x, g), gh)
        torch.autograd.grad(h, (x, g), gh)
    # the explicit pair in a graph, replayed with other gradients
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.linear_recurrence_bwd(res, (gh, None))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = kernels.linear_recurrence_bwd(res, (gh, None))
    for _ in range(3):
        gh.copy_(torch.randn(2, T, 136, device="cuda"))
        want = kernels.linear_recurrence_bwd(res, (gh, None))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(outs, want)
