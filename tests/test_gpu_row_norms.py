"""The gated norm and the residual norm on the GPU, against the 64-bit forms.

Tolerances: half a step of the output's type relative to its value (bf16 2^-8, fp32 2^-24), and fp32
arithmetic: a row's sum over C terms is off by at most C / 256 + 16 additions of 2^-24 (each lane adds
its own, then the lanes), its root half of that; the exponential and reciprocal of the gate 2^-22 each
(its argument is rounded: |z| 2^-24 more); a dozen operations of 2^-24 beside. An output without
differences is off by (C / 256 + 128) 2^-24 of its value. A gradient is a difference, r (p - n mean(p n)),
whose two terms may all but cancel (in a row of one element they do): each of them is computed to
(C / 256 + 128) 2^-24 of itself, so the difference is off by that of the sum of their absolute values,
which ``gated_bwd_size`` and ``residual_bwd_size`` give, and so are sums over rows, which add fp32's
(rows) 2^-24 of the sum of absolute values. h is a sum of two terms: relative to both.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import decay_oracle as ref
from prometheus_amd import kernels

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
WIDTHS = [1, 7, 32, 33, 64, 100, 128, 192, 256, 500, 1001, 1024, 2000, 2560, 4096, 5000, 8192, 10000, 16384]


def normal(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def near_rows(got, want, C, size=None):
    rnd = torch.finfo(got.dtype).eps / 2
    off = (got.detach().cpu().double() - want).abs()
    size = want.abs().amax(-1, keepdim=True) if size is None else size.amax(-1, keepdim=True)
    allowed = rnd * want.abs() + (C / 256 + 128) * 2.0**-24 * size + 1e-37
    assert got.shape == want.shape and bool((off <= allowed).all()), (off / allowed).max().item()


def near_sums(got, want, size, rows, C):
    off = (got.detach().cpu().double() - want).abs()
    allowed = (rows + C / 256 + 128) * 2.0**-24 * size + 1e-37
    assert got.dtype == F32 and got.shape == want.shape and bool((off <= allowed).all()), (off / allowed).max().item()


def check_gated(x, z, w, gy, options, y, grads):
    C, rows = x.shape[-1], x.numel() // x.shape[-1]
    near_rows(y, ref.gated(x, z, w, **options), C)
    want = ref.gradients(lambda *a: ref.gated(*a, **options), (x, z, w), (gy,))
    size = ref.gated_bwd_size(x, z, w, gy, **options)
    near_rows(grads[0], want[0], C, size[0])
    near_rows(grads[1], want[1], C, size[1])
    if w is not None:
        near_sums(grads[2], want[2], size[2], rows, C)


@pytest.mark.parametrize("types", [(BF16, BF16), (F32, F32), (F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("C", WIDTHS)
def test_gated(C, types):
    xt, zt = types
    options = {"activation": "silu" if C % 2 else "sigmoid", "gate_first": C in (7, 128, 2000, 8192)}
    x, z, gy = (normal(5, 3, C, seed=i).to(t) for i, t in enumerate((xt, zt, xt)))
    w = (1 + 0.1 * normal(C, seed=4)).to(zt)
    dev = [t.cuda().requires_grad_(True) for t in (x, z, w)]
    y = kernels.gated_norm(*dev, **options)
    grads = torch.autograd.grad(y, dev, gy.cuda())
    assert [g.dtype for g in grads] == [xt, zt, zt] and y.dtype == xt
    _, res = kernels.gated_norm_fwd(*(t.detach() for t in dev), **options)
    gw = kernels.gated_norm_bwd(res, gy.cuda())[2]  # (in fp32)
    check_gated(x, z, w, gy, options, y, [grads[0], grads[1], gw])
    assert torch.equal(grads[2], gw.to(zt))


@pytest.mark.parametrize("activation", ["silu", "sigmoid"])
@pytest.mark.parametrize("gate_first", [False, True])
@pytest.mark.parametrize("C", [64, 3000])
def test_gated_forms(activation, gate_first, C):
    options = {"activation": activation, "gate_first": gate_first}
    x, z, gy = (normal(9, C, seed=i) for i in range(3))
    dev = [t.cuda() for t in (x, z)]
    y, res = kernels.gated_norm_fwd(*dev, **options)
    gx, gz, gw = kernels.gated_norm_bwd(res, gy.cuda())
    assert gw is None
    check_gated(x, z, None, gy, options, y, (gx, gz))


def test_gated_views():
    """Gates that are a part of a projection, heads moved, odd offsets: the same bits as copies."""
    B, T, H, C = 2, 5, 3, 64
    wide = normal(B, T, 2 * H, C).to(BF16).cuda()
    x = normal(B, H, T, C, seed=1).to(BF16).cuda().transpose(1, 2)
    odd = torch.zeros(B, T, H, C + 3, dtype=BF16, device="cuda")[..., 1:1 + C]
    odd.copy_(wide[:, :, H:])
    w = 1 + 0.1 * normal(C, seed=2).cuda()
    want, res = kernels.gated_norm_fwd(x.contiguous(), wide[:, :, H:].contiguous(), w)
    gy = torch.randn_like(want)
    grads = kernels.gated_norm_bwd(res, gy)
    for z in (wide[:, :, H:], odd):
        y, r = kernels.gated_norm_fwd(x, z, w)
        assert torch.equal(y, want)
        assert all(torch.equal(a, b) for a, b in zip(kernels.gated_norm_bwd(r, gy), grads))


def test_gated_many_rows():
    """More rows than workgroups stay on the card: each walks through several."""
    x, z, gy = (normal(70001, 64, seed=i).to(BF16).cuda() for i in range(3))
    w = 1 + 0.1 * normal(64, seed=4).cuda()
    y, res = kernels.gated_norm_fwd(x, z, w)
    gx, gz, gw = kernels.gated_norm_bwd(res, gy)
    xd, zd, gd, wd = (t.double() for t in (x, z, gy, w))
    near_rows(y, ref.gated(xd, zd, wd).cpu(), 64)
    ex, ez, ew = (t.cpu() for t in ref.gradients(ref.gated, (xd, zd, wd), (gd,)))
    size = [t.cpu() for t in ref.gated_bwd_size(xd, zd, wd, gd)]
    near_rows(gx, ex, 64, size[0])
    near_rows(gz, ez, 64, size[1])
    near_sums(gw, ew, size[2], 70001, 64)
    assert torch.equal(kernels.gated_norm_bwd(res, gy)[2], gw)


def check_residual(x, r, w, wp, gy, gh, scale, out, grads):
    C, rows = x.shape[-1], x.numel() // x.shape[-1]

    def f(x, r, w, wp):
        return ref.residual(x, r, w, wp, scale)

    y, h = f(x, r, w, wp)
    terms = r.double().abs() + (h - r.double()).abs()  # of h
    near_rows(out[0], y, C, y.abs() + terms * (y / h).nan_to_num().abs().amax(-1, keepdim=True))
    near_rows(out[1], h, C, terms)
    want = ref.gradients(f, (x, r, w, wp), (gy, gh))
    size = ref.residual_bwd_size(x, r, w, wp, gy, gh, scale)
    # (n = r h too is off by its terms' size: where h's own nearly cancel, by more of itself)
    worse = 1 + (terms.square().sum(-1, keepdim=True) / h.square().sum(-1, keepdim=True)).sqrt()
    near_rows(grads[0], want[0], C, 2 * worse * size[0])
    near_rows(grads[1], want[1], C, 2 * worse * size[1])
    for i in (2, 3):
        if want[i] is not None:
            near_sums(grads[i], want[i], 2 * worse.max() * size[i], rows, C)


@pytest.mark.parametrize("types", [(BF16, BF16), (F32, F32), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("C", WIDTHS)
def test_residual(C, types):
    xt, rt = types
    post, scale = C % 3 != 0, 0.5 if C % 2 else 1.0
    x, r, gy, gh = (normal(7, C, seed=i).to(t) for i, t in enumerate((xt, rt, xt, rt)))
    w = 1 + 0.1 * normal(C, seed=5)
    wp = 1 + 0.1 * normal(C, seed=6) if post else None
    dev = [None if t is None else t.cuda().requires_grad_(True) for t in (x, r, w, wp)]
    out = kernels.residual_norm(*dev[:3], post_weight=dev[3], scale=scale)
    grads = torch.autograd.grad(out, [t for t in dev if t is not None], (gy.cuda(), gh.cuda()))
    assert out[0].dtype == xt and out[1].dtype == rt and grads[0].dtype == xt and grads[1].dtype == rt
    check_residual(x, r, w, wp, gy, gh, scale, out, [*grads, None])


def test_residual_missing_gradients_and_weights():
    x, r, gy = (normal(4, 6, 96, seed=i).cuda() for i in range(3))
    (y, h), res = kernels.residual_norm_fwd(x, r)
    zero = torch.zeros_like(gy)
    for grads, full in (((gy, None), (gy, zero)), ((None, gy), (zero, gy))):
        got, want = kernels.residual_norm_bwd(res, grads), kernels.residual_norm_bwd(res, full)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[2] is None and got[3] is None
    check_residual(*(t.cpu() for t in (x, r)), None, None, gy.cpu(), zero.cpu(), 1.0, (y, h),
                   kernels.residual_norm_bwd(res, (gy, zero)))


def test_residual_views_and_weights_types():
    x = normal(3, 8, 200).to(BF16).cuda()[:, ::2, 3:131]
    r = normal(3, 4, 128, seed=1).cuda().transpose(0, 1).contiguous().transpose(0, 1)
    w, wp = (1 + 0.1 * normal(128, seed=2)).to(BF16).cuda(), 1 + 0.1 * normal(128, seed=3).cuda()
    got = kernels.residual_norm(x, r, w, post_weight=wp)
    want = kernels.residual_norm(x.contiguous(), r.contiguous(), w.float(), post_weight=wp)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_zeros_and_extremes():
    """Rows of zeros, closed and wide open gates, infinities in their own row only."""
    x, z = torch.zeros(3, 64).cuda(), normal(3, 64).cuda()
    assert not kernels.gated_norm(x, z).any()
    z[0] = -1e4
    z[1] = 1e4
    y = kernels.gated_norm(normal(3, 64, seed=1).cuda(), z)
    assert not y[0].any() and torch.isfinite(y).all()
    y, res = kernels.gated_norm_fwd(normal(3, 64, seed=1).cuda(), z)
    assert all(torch.isfinite(g).all() for g in kernels.gated_norm_bwd(res, torch.ones_like(y))[:2])
    x[1] = float("inf")
    y, h = kernels.residual_norm(x, torch.ones_like(x))
    assert torch.isfinite(y[[0, 2]]).all() and torch.isinf(h[1]).all()


def test_no_rows():
    x = torch.zeros(0, 5, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    y, res = kernels.gated_norm_fwd(x, x, w)
    assert y.shape == x.shape and not kernels.gated_norm_bwd(res, y)[2].any()
    (y, h), res = kernels.residual_norm_fwd(x, x, w, post_weight=w)
    grads = kernels.residual_norm_bwd(res, (y, h))
    assert h.shape == x.shape and not grads[2].any() and not grads[3].any()


def test_hosts():
    x, z = normal(3, 64).numpy(), normal(3, 64, seed=1).numpy()
    y = kernels.gated_norm(x, z)
    assert isinstance(y, np.ndarray)
    near_rows(torch.from_numpy(y), ref.gated(torch.from_numpy(x), torch.from_numpy(z)), 64)
    y, h = kernels.residual_norm(torch.from_numpy(x), torch.from_numpy(z))
    assert y.device.type == "cpu" and h.device.type == "cpu"


def test_graph_replays():
    x, z, r, gy = (normal(40, 256, seed=i).to(BF16).cuda() for i in range(4))
    w = 1 + 0.1 * normal(256, seed=5).cuda()

    def step():
        y, a = kernels.gated_norm_fwd(x, z, w)
        (u, h), b = kernels.residual_norm_fwd(y, r, w, post_weight=w)
        grads = kernels.residual_norm_bwd(b, (gy, gy))
        return y, u, h, *grads, *kernels.gated_norm_bwd(a, grads[0])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        for j, t in enumerate((x, z, r, gy)):
            t.copy_(normal(40, 256, seed=20 + 4 * i + j))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_saved_tensors_may_come_back_elsewhere():
    x, z, gy = (normal(4, 6, 96, seed=i).to(BF16) for i in range(3))
    w = 1 + 0.1 * normal(96, seed=3)

    def grads(pack, unpack):
        dev = [t.cuda().requires_grad_(True) for t in (x, z, w)]
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            y = kernels.gated_norm(*dev)
            out = kernels.residual_norm(y, dev[1], dev[2], post_weight=dev[2])
        return torch.autograd.grad(out, dev, (gy.cuda(), gy.cuda()))

    want = grads(lambda t: t, lambda t: t)
    for unpack in (lambda t: t, lambda t: t.cuda().t().contiguous().t() if t.dim() == 2 else t.cuda()):
        got = grads(lambda t: t.cpu(), unpack)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_of_what_is_asked_for():
    x, z = (normal(5, 64, seed=i).cuda() for i in range(2))
    w = (1 + 0.1 * normal(64, seed=3)).cuda().requires_grad_(True)
    gw, = torch.autograd.grad(kernels.gated_norm(x, z, w).sum(), w)
    gx, = torch.autograd.grad(kernels.gated_norm(x.requires_grad_(True), z, w.detach()).sum(), x)
    assert gw.shape == (64,) and gx.shape == x.shape
    y, h = kernels.residual_norm(x.detach(), z, w, post_weight=w)
    g, = torch.autograd.grad(y.sum(), w)  # (one weight in both places: its gradients add)
    a, b = (w.detach().clone().requires_grad_(True) for _ in range(2))
    both = torch.autograd.grad(kernels.residual_norm(x.detach(), z, a, post_weight=b)[0].sum(), (a, b))
    assert torch.allclose(g, both[0] + both[1], rtol=1e-6)


def test_fp16_and_fp64_run_in_fp32():
    x, z = normal(5, 64), normal(5, 64, seed=1)
    want = kernels.gated_norm(x.cuda(), z.cuda())
    d = [t.cuda().double().requires_grad_(True) for t in (x, z)]
    y = kernels.gated_norm(*d)
    assert y.dtype == F32 and torch.equal(y, want)
    assert all(g.dtype == torch.float64 for g in torch.autograd.grad(y.sum(), d))


@pytest.mark.parametrize("C", [128, 4096])
def test_another_stream(C):
    x, z = (normal(300, C, seed=i).cuda() for i in range(2))
    want = kernels.residual_norm(x, z)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernels.residual_norm(x, z)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits():
    rows, C = (1 << 19) + 3, 4100  # 2.1e9 elements a tensor
    x, z, gy, gh = (torch.empty(rows, C, dtype=torch.bfloat16, device="cuda").normal_() for _ in range(4))
    last = slice(rows - 5, rows)
    y, res = kernels.gated_norm_fwd(x, z)
    want, res2 = kernels.gated_norm_fwd(x[last], z[last])
    assert torch.equal(y[last], want)
    for a, b in zip(kernels.gated_norm_bwd(res, gy)[:2], kernels.gated_norm_bwd(res2, gy[last])):
        assert torch.equal(a[last], b)
    (y, h), res = kernels.residual_norm_fwd(x, z)
    (want_y, want_h), res2 = kernels.residual_norm_fwd(x[last], z[last])
    assert torch.equal(y[last], want_y) and torch.equal(h[last], want_h)
    for a, b in zip(kernels.residual_norm_bwd(res, (gy, gh))[:2], kernels.residual_norm_bwd(res2, (gy[last], gh[last]))):
        assert torch.equal(a[last], b)
