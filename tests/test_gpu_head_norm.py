"""GPU tests of the heads' norms with the position rotation against their 64-bit form.

Tolerances are the oracle's error bounds for fp32 arithmetic plus half a step of the output's
type, per element.
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


def _check(q, k, table, pos, norm, wq, wk, interleaved, eps=1e-6, grads=(True, True)):
    """Forward and backward of one call against the oracle."""
    opts = dict(norm=norm, q_weight=wq, k_weight=wk, interleaved=interleaved, eps=eps)
    outs, res = kernels.norm_rotate_fwd(q, k, table, pos, **opts)
    plain = kernels.norm_rotate(q, k, table, pos, **opts)
    assert all(torch.equal(a, b) for a, b in zip(outs, plain))
    hpos = None
    if table is not None:
        hpos = np.broadcast_to(np.arange(q.shape[1]) if pos is None else pos.cpu().numpy(), q.shape[:-2])
    gz = [torch.randn(x.shape, device="cuda").to(outs[0].dtype) if want else None for x, want in zip((q, k), grads)]
    got = kernels.norm_rotate_bwd(res, gz)
    assert all(a is None or torch.equal(a, b) for a, b in zip(got, kernels.norm_rotate_bwd(res, gz)))
    for i, (x, w) in enumerate(((q, wq), (k, wk))):
        a = (_host(x), _host(table), hpos, norm, _host(w), eps, interleaved)
        _near(outs[i], ref.head_norm(*a), ref.head_norm_bound(*a), "qk"[i])
        g = np.zeros(x.shape) if gz[i] is None else _host(gz[i])
        b = (a[0], g, *a[1:])
        want, bound = ref.head_norm_bwd(*b), ref.head_norm_bwd_bound(*b)
        _near(got[i], want[0], bound[0], ("gq", "gk")[i])
        if w is None:
            assert got[2 + i] is None
        else:
            assert got[2 + i].dtype == F32
            _near(got[2 + i], want[1], bound[1], ("gwq", "gwk")[i])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("norm", ["l2", "rms"])
@pytest.mark.parametrize("D,R", [(1, 0), (2, 2), (5, 4), (33, 32), (64, 64), (64, 0), (80, 40), (96, 96), (128, 128),
                                 (128, 64), (128, 6), (192, 96), (250, 250), (256, 256)])
def test_sizes(D, R, norm, dtype):
    rng = torch.Generator(device="cuda").manual_seed(D + R)
    B, T, Hq, Hk = 2, 5, 6, 3
    for interleaved in (False, True):
        for weight in (False, True):
            q = torch.randn(B, T, Hq, D, generator=rng, device="cuda").to(dtype)
            k = torch.randn(B, T, Hk, D, generator=rng, device="cuda").to(dtype)
            table = kernels.rotation_table(T + 3, R) if R else None
            pos = torch.randint(0, T + 3, (B, T), generator=rng, device="cuda") if R and weight else None
            ws = [1 + 0.3 * torch.randn(D, generator=rng, device="cuda") if weight else None for _ in range(2)]
            _check(q, k, table, pos, norm, *ws, interleaved)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,Hq,Hk,D", [(1, 1, 1, 1, 128), (3, 1, 32, 8, 128), (1, 1000, 4, 4, 64), (2, 77, 16, 1, 96),
                                         (5, 3, 7, 5, 256), (1, 700, 24, 24, 128)])
def test_batches(B, T, Hq, Hk, D, dtype):
    q, k = (torch.randn(B, T, H, D, device="cuda").to(dtype) for H in (Hq, Hk))
    w = 1 + 0.1 * torch.randn(D, device="cuda")
    _check(q, k, kernels.rotation_table(T, D), None, "rms", w, None, False)
    _check(q, k, kernels.rotation_table(T, D), None, "l2", None, w.to(BF16), True, grads=(True, False))
    _check(q, k, None, None, "l2", None, None, False, grads=(False, True))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_single_tokens_at_any_position(dtype):
    N, H, D = 50, 8, 128
    table = kernels.rotation_table(40000, D)
    pos = torch.randint(0, 40000, (N,), device="cuda")
    q, k = (torch.randn(N, H, D, device="cuda").to(dtype) for _ in range(2))
    want = kernels.norm_rotate(q[None], k[None], table, pos[None])
    for p in (pos, pos.int(), pos.cpu(), pos.cpu().numpy()):
        got = kernels.norm_rotate(q, k, table, p)
        assert all(torch.equal(a, b[0]) for a, b in zip(got, want))
    hp = pos.cpu().numpy()
    a = (_host(q), _host(table), hp)
    _near(got[0], ref.head_norm(*a), ref.head_norm_bound(*a), "q")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [48, 128])
def test_views_are_read_in_place(D, dtype):
    B, T, Hq, Hk = 2, 9, 4, 2
    qkv = torch.randn(B, T, (Hq + 2 * Hk) * D + 3, device="cuda").to(dtype)
    table = kernels.rotation_table(T, D)
    for off in (0, 1, 3):
        flat = qkv[..., off:off + (Hq + 2 * Hk) * D].unflatten(-1, (-1, D))
        q, k = flat[:, :, :Hq], flat[:, :, Hq:Hq + Hk]
        cases = [(q, k), (q.transpose(1, 2).contiguous().transpose(1, 2), k), (q[:, :, :1].expand(B, T, Hq, D), k),
                 (q.transpose(2, 3).contiguous().transpose(2, 3), k), (q[:1].expand(B, T, Hq, D), k)]
        for a, b in cases:
            want, res = kernels.norm_rotate_fwd(a.contiguous(), b.contiguous(), table)
            got, res2 = kernels.norm_rotate_fwd(a, b, table)
            assert all(torch.equal(u, v) for u, v in zip(got, want))
            gz = [torch.randn(x.shape, device="cuda").to(dtype) for x in (a, b)]
            for u, v in zip(kernels.norm_rotate_bwd(res2, gz)[:2], kernels.norm_rotate_bwd(res, gz)[:2]):
                assert torch.equal(u, v)


def test_positions_of_every_layout():
    B, T, H, D = 3, 6, 2, 64
    q, k = (torch.randn(B, T, H, D, device="cuda") for _ in range(2))
    table = kernels.rotation_table(50, D)
    p = torch.randint(0, 50, (B, T), device="cuda")
    want = kernels.norm_rotate(q, k, table, p)
    wide = torch.zeros(B, 2 * T, dtype=torch.int64, device="cuda")
    wide[:, :T] = p
    for other in (p.int(), wide[:, :T], p.t().contiguous().t(), p.cpu()):
        assert all(torch.equal(a, b) for a, b in zip(kernels.norm_rotate(q, k, table, other), want))
    row = kernels.norm_rotate(q, k, table, p[0])
    same = kernels.norm_rotate(q, k, table, p[:1].expand(B, T))
    assert all(torch.equal(a, b) for a, b in zip(row, same))
    none = kernels.norm_rotate(q, k, table)
    count = kernels.norm_rotate(q, k, table, torch.arange(T, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(none, count))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D,R", [(128, 128), (128, 64), (40, 6)])
def test_positions_outside_the_table_are_nan_rows(D, R, dtype):
    N, H = 6, 3
    table = kernels.rotation_table(10, R)
    q, k = (torch.randn(N, H, D, device="cuda").to(dtype) for _ in range(2))
    pos = torch.tensor([0, 10, -1, 9, 2**40, 3], device="cuda")
    bad = torch.tensor([False, True, True, False, True, False], device="cuda")
    outs, res = kernels.norm_rotate_fwd(q, k, table, pos)
    good = kernels.norm_rotate(q[~bad], k[~bad], table, pos[~bad])
    grads = kernels.norm_rotate_bwd(res, outs)
    for o, w, g in zip(outs, good, grads):
        assert torch.isnan(o[bad]).all() and torch.equal(o[~bad], w)
        assert torch.isnan(g[bad]).all() and torch.isfinite(g[~bad]).all()


def test_rows_of_zeros_infinities_and_nan():
    q = torch.randn(1, 8, 2, 128, device="cuda")
    q[0, 1] = 0.0
    q[0, 2] *= 1e-9  # below eps
    q[0, 3, 0, 5] = torch.nan
    q[0, 4, 0, 5] = torch.inf
    k = q.clone()
    for norm in ("l2", "rms"):
        for dtype in (F32, BF16):
            (zq, zk), res = kernels.norm_rotate_fwd(q.to(dtype), k.to(dtype), norm=norm)
            assert not zq[0, 1].any()
            assert torch.isnan(zq[0, 3, 0]).all() and torch.isfinite(zq[0, 3, 1]).all()
            assert torch.isnan(zq[0, 4, 0, 5]) and (zq[0, 4, 0, :5] == 0).all()
            assert torch.isfinite(zq[0, [0, 1, 2, 5, 6, 7]]).all()
            gz = torch.randn_like(zq)
            gq = kernels.norm_rotate_bwd(res, (gz, None))[0]
            hq = _host(q.to(dtype))[:, [0, 1, 2, 5]]
            a = (hq, _host(gz)[:, [0, 1, 2, 5]], None, None, norm)
            _near(gq[:, [0, 1, 2, 5]], ref.head_norm_bwd(*a)[0], ref.head_norm_bwd_bound(*a)[0], norm)
            assert torch.isnan(gq[0, 3, 0]).all() and torch.isfinite(gq[0, 3, 1]).all()


def test_no_rows():
    for B, T in ((0, 4), (2, 0)):
        q, k = torch.empty(B, T, 4, 64, device="cuda"), torch.empty(B, T, 2, 64, device="cuda")
        w = torch.ones(64, device="cuda")
        (zq, zk), res = kernels.norm_rotate_fwd(q, k, kernels.rotation_table(4, 64), q_weight=w)
        assert zq.shape == q.shape and zk.shape == k.shape
        gq, gk, gwq, gwk = kernels.norm_rotate_bwd(res, (zq, zk))
        assert gq.shape == q.shape and gwk is None and torch.equal(gwq, torch.zeros(64, device="cuda"))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_autograd(dtype):
    B, T, Hq, Hk, D = 2, 40, 6, 2, 96
    q, k = (torch.randn(B, T, H, D, device="cuda").to(dtype).requires_grad_(True) for H in (Hq, Hk))
    wq = (1 + 0.1 * torch.randn(D, device="cuda")).to(dtype).requires_grad_(True)
    wk = (1 + 0.1 * torch.randn(D, device="cuda")).to(dtype).requires_grad_(True)
    table = kernels.rotation_table(T, 48)
    zq, zk = kernels.norm_rotate(q, k, table, norm="rms", q_weight=wq, k_weight=wk)
    gq, gk = torch.randn_like(zq), torch.randn_like(zk)
    got = torch.autograd.grad((zq, zk), (q, k, wq, wk), (gq, gk), retain_graph=True)
    assert [t.dtype for t in got] == [dtype] * 4
    pos = np.broadcast_to(np.arange(T), (B, T))
    for i, (x, w, gz) in enumerate(((q, wq, gq), (k, wk, gk))):
        a = (_host(x), _host(gz), _host(table), pos, "rms", _host(w))
        want, bound = ref.head_norm_bwd(*a), ref.head_norm_bwd_bound(*a)
        _near(got[i], want[0], bound[0], i)
        _near(got[2 + i], want[1], bound[1], i)
    (only,) = torch.autograd.grad(zk, k, gk)  # q's output unused, no weights wanted
    assert torch.equal(only, got[1])
    # fp32 weights beside bf16 heads, and mixed ones
    w32 = wq.detach().float().requires_grad_(True)
    zq, _ = kernels.norm_rotate(q, k, table, norm="rms", q_weight=w32, k_weight=wk)
    (gw,) = torch.autograd.grad(zq, w32, gq)
    assert gw.dtype == F32


def test_gradients_against_differences():
    """Along a direction, differences of the kernel's own fp32 forward."""
    q, k = (torch.randn(1, 7, 3, 64, device="cuda") for _ in range(2))
    w = 1 + 0.1 * torch.randn(64, device="cuda")
    table = kernels.rotation_table(7, 64)
    gz = torch.randn_like(q)
    for norm in ("l2", "rms"):
        _, res = kernels.norm_rotate_fwd(q, k, table, norm=norm, q_weight=w)
        gq, _, gw, _ = kernels.norm_rotate_bwd(res, (gz, None))
        e = 2.0**-8
        pos = np.broadcast_to(np.arange(7), (1, 7))
        noise = 2 * np.sum(np.abs(_host(gz)) * ref.head_norm_bound(_host(q), _host(table), pos, norm, _host(w))) / e
        for at, grad in ((0, gq), (1, gw)):
            v = torch.randn_like(grad)
            side = []
            for s in (2, 1, -1, -2):
                args = [q, w]
                args[at] = args[at] + s * e * v
                z = kernels.norm_rotate(args[0], k, table, norm=norm, q_weight=args[1])[0]
                side.append(float((gz.double() * z.double()).sum()))
            wide, near = (side[0] - side[3]) / (4 * e), (side[1] - side[2]) / (2 * e)
            assert abs(near - float((grad.double() * v.double()).sum())) <= noise + abs(wide - near)


def test_host_arrays():
    rng = np.random.default_rng(0)
    q, k = rng.normal(size=(2, 5, 3, 16)).astype(np.float32), rng.normal(size=(2, 5, 1, 16)).astype(np.float32)
    table = kernels.rotation_table(5, 16)
    zq, zk = kernels.norm_rotate(q, k)
    assert isinstance(zq, np.ndarray)
    np.testing.assert_allclose(zk, ref.head_norm(k), rtol=1e-5, atol=1e-6)
    zq, zk = kernels.norm_rotate(torch.from_numpy(q), torch.from_numpy(k), table.cpu())
    assert zq.device.type == "cpu"
    pos = np.broadcast_to(np.arange(5), (2, 5))
    np.testing.assert_allclose(zq.numpy(), ref.head_norm(q, _host(table), pos), rtol=1e-4, atol=1e-5)


def test_another_stream_and_graph_replays():
    B, H, D = 32, 8, 128
    table = kernels.rotation_table(1000, D)
    pos = torch.zeros(B, dtype=torch.int32, device="cuda")
    q, k = (torch.randn(B, H, D, device="cuda").to(BF16) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernels.norm_rotate(q, k, table, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, kernels.norm_rotate(q, k, table, pos)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = kernels.norm_rotate(q, k, table, pos)
    for i in range(4):
        pos.copy_(torch.randint(0, 1000, (B,)))
        q.copy_(torch.randn(B, H, D))
        want = kernels.norm_rotate(q, k, table, pos)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
