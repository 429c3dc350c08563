"""GPU tests of the operators beside the delta rule where their ranges end: the most heads, offsets
and tables that stand for nothing, saved tensors that come back changed, states without bound."""

from __future__ import annotations

import pytest
import torch

from prometheus_amd import kernels, serving

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def test_the_most_heads():
    """2^24 heads of 256: a head's offset inside its token passes 31 bits. The same bits as in calls
    of a few heads, forward and backward."""
    H, D, cut = 2**24 - 1, 256, 2**22
    q = torch.randn(1, H, D, dtype=BF16, device="cuda")
    k = q[:, :1].contiguous()
    (zq, zk), res = kernels.norm_rotate_fwd(q, k)
    gq, gk, _, _ = kernels.norm_rotate_bwd(res, (zq, zk))
    assert torch.equal(zk, zq[:, :1]) and torch.equal(gk, gq[:, :1])
    for a in range(0, H, cut):
        part = q[:, a:a + cut]
        (want, _), res = kernels.norm_rotate_fwd(part, k)
        assert torch.equal(zq[:, a:a + cut], want), a
        assert torch.equal(gq[:, a:a + cut], kernels.norm_rotate_bwd(res, (want, None))[0]), a


def _recurrence_step():
    x, g = torch.randn(2, 300, 24, device="cuda").to(BF16), (-torch.rand(2, 300, 24, device="cuda")).to(BF16)
    return kernels.linear_recurrence, [x, g, torch.randn(2, 24, device="cuda")]


def _heads_step():
    q, k = (torch.randn(2, 9, h, 64, device="cuda").to(BF16) for h in (4, 2))
    table = kernels.rotation_table(9, 32)
    w = 1 + 0.1 * torch.randn(64, device="cuda")
    return lambda q, k, w: kernels.norm_rotate(q, k, table, torch.arange(9, device="cuda"), q_weight=w), [q, k, w]


@pytest.mark.parametrize("step", [_recurrence_step, _heads_step])
def test_saved_tensors_that_come_back_changed(step):
    """On the host, in a wider type, with other strides, with fewer rows."""
    f, args = step()
    args = [t.requires_grad_(True) for t in args]

    def grads(pack, unpack):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            a, b = f(*args)
        return torch.autograd.grad(a.float().square().sum() + b.float().sum(), args)

    def same(t):
        return t

    def wide(t):
        return t.double() if t.is_floating_point() else t.int()

    def turned(t):
        return t.transpose(0, -1).contiguous().transpose(0, -1)

    want = grads(same, same)
    for pack, unpack in ((torch.Tensor.cpu, same), (wide, same), (turned, same), (lambda t: turned(wide(t)).cpu(), same)):
        assert all(torch.equal(a, b) for a, b in zip(grads(pack, unpack), want))
    with pytest.raises(kernels.KernelError):
        grads(same, lambda t: t[:-1])


@pytest.mark.parametrize("cu", [[0, 2**32 + 100, 400], [2**32, 100, 400], [0, 100, 2**32 + 400], [0, 100 - 2**32, 400]])
def test_wide_offsets_do_not_come_back_into_range(cu):
    """64-bit offsets on the GPU whose lower halves are good ones."""
    N, C = 400, 16
    x, g = torch.randn(N, C, device="cuda"), -torch.rand(N, C, device="cuda")
    offsets = torch.tensor(cu, device="cuda")
    kernels.linear_recurrence_varlen(x, g, offsets)
    with pytest.raises(kernels.KernelError):
        kernels.check_varlen()
    cache = serving.RecurrenceStateCache(1, 2, C)
    cache.prefill(0, torch.tensor([0, 1], device="cuda"), x, g, offsets)
    with pytest.raises(kernels.KernelError):
        kernels.check_varlen()
    kernels.linear_recurrence_varlen(x[:0], g[:0], offsets[:1])  # (launches nothing: checked apart)
    if cu[0]:
        with pytest.raises(kernels.KernelError):
            kernels.check_varlen()
    q, k, v = (torch.randn(N, 1, 64, device="cuda") for _ in range(3))
    kernels.chunked_delta_rule_varlen(q, k, v, torch.rand(N, 1, device="cuda"), offsets)
    with pytest.raises(kernels.KernelError):
        kernels.check_varlen()
    good = torch.tensor([0, 100, 400], device="cuda")
    want = kernels.linear_recurrence_varlen(x, g, good.int())
    assert all(torch.equal(a, b) for a, b in zip(kernels.linear_recurrence_varlen(x, g, good), want))
    kernels.check_varlen()


@pytest.mark.parametrize("interleaved", [False, True])
def test_a_table_without_rows(interleaved):
    """No tokens need none of it; a token at any position is outside it, and comes out as NaN."""
    table, w = kernels.rotation_table(0, 64), torch.ones(64, device="cuda")
    assert table.shape == (0, 64)
    q, k = torch.empty(2, 0, 4, 64, device="cuda"), torch.empty(2, 0, 2, 64, device="cuda")
    (zq, zk), res = kernels.norm_rotate_fwd(q, k, table, q_weight=w, interleaved=interleaved)
    gq, gk, gw, _ = kernels.norm_rotate_bwd(res, (zq, zk))
    assert zq.shape == gq.shape == q.shape and zk.shape == gk.shape == k.shape and not gw.any()
    q, k = torch.randn(3, 4, 64, device="cuda"), torch.randn(3, 2, 64, device="cuda")
    outs, res = kernels.norm_rotate_fwd(q, k, table, torch.tensor([0, -1, 5], device="cuda"), interleaved=interleaved)
    grads = kernels.norm_rotate_bwd(res, outs)[:2]
    assert all(torch.isnan(t).all() for t in (*outs, *grads))
    with pytest.raises(kernels.KernelError):
        kernels.norm_rotate(q, k, table, [0, 1, 2], interleaved=interleaved)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [1, 100, 256, 700, 9000, 20000])
def test_an_infinite_state_passes_open_gates(T, dtype):
    """Gates of exp(-2), whose products over a span are zero in fp32: what is infinite stays so, from
    the initial state, from a token, packed, and back from the last gradient."""
    C = 70
    x, g = torch.randn(2, T, C, device="cuda").to(dtype), torch.full((2, T, C), -2.0, dtype=dtype, device="cuda")
    g[:, :, 1::4] = -40.0  # (the products of a few tokens are)
    s0 = torch.randn(2, C, device="cuda")
    inf, at = torch.inf, T // 3
    hit = torch.zeros(2, T, C, device="cuda")
    s0[0, 5], s0[1, 8] = inf, -inf
    x[1, at, 13], x[0, at, 16] = inf, -inf
    hit[0, :, 5], hit[1, :, 8], hit[1, at:, 13], hit[0, at:, 16] = inf, -inf, inf, -inf
    still = hit == 0
    end = hit[:, -1] != 0

    def check(h, s):
        assert torch.equal(h[~still].float(), hit[~still]) and torch.isfinite(h[still]).all()
        assert torch.equal(s[end], hit[:, -1][end]) and torch.isfinite(s[~end]).all()

    (h, s), res = kernels.linear_recurrence_fwd(x, g, s0, out_dtype=dtype)
    check(h, s)
    cu = torch.tensor([0, T, 2 * T], device="cuda")
    h, s = kernels.linear_recurrence_varlen(x.reshape(2 * T, C), g.reshape(2 * T, C), cu, s0, out_dtype=dtype)
    check(h.reshape(2, T, C), s)
    clean = torch.randn(2, T, C, device="cuda").to(dtype), torch.randn(2, C, device="cuda")
    _, res = kernels.linear_recurrence_fwd(clean[0], g, clean[1], out_dtype=dtype)
    gh, gs = torch.randn(2, T, C, device="cuda").to(dtype), torch.randn(2, C, device="cuda")
    gs[0, 5], gh[1, at, 9] = inf, -inf
    gx, gg, gs0 = kernels.linear_recurrence_bwd(res, (gh, gs))
    hit = torch.zeros(2, T, C, device="cuda")
    hit[0, :, 5], hit[1, :at + 1, 9] = inf, -inf
    still = hit == 0
    assert torch.equal(gx[~still].float(), hit[~still]) and torch.isfinite(gx[still]).all()
    assert gs0[0, 5] == inf and gs0[1, 9] == -inf and torch.isfinite(gg[still]).all()
    assert torch.isinf(gg[~still]).all()  # (h before each token is not zero here)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [40, 700, 9000])
def test_a_closed_gate_leaves_nothing(T, dtype):
    """exp(-inf) is zero, whatever its neighbours: a finite state before it is gone to the last bit."""
    x, g = torch.zeros(1, T, 66, dtype=dtype, device="cuda"), torch.full((1, T, 66), -3.0, dtype=dtype, device="cuda")
    g[0, T // 2] = -torch.inf
    s0 = torch.full((1, 66), 1e38, device="cuda")
    (h, s), res = kernels.linear_recurrence_fwd(x, g, s0, out_dtype=dtype)
    assert not h[0, T // 2:].any() and not s.any() and h[0, :T // 2].float()[:10].all()
    gx, _, gs0 = kernels.linear_recurrence_bwd(res, (None, s0))
    assert not gx[0, :T // 2].any() and not gs0.any()
