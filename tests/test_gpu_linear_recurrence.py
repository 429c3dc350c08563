"""GPU tests of the elementwise gated linear recurrence against its 64-bit form.

Tolerances are the oracle's error bounds for fp32 arithmetic (the roundings on each term's way)
plus half a step of the output's type, per element.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import layer_oracle as ref
from prometheus_amd import kernels, serving

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
TYPES = [(BF16, BF16, BF16), (BF16, F32, BF16), (BF16, BF16, F32), (F32, F32, F32), (F32, F32, BF16)]


def _host(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _near(got, want, bound, name, rows=None):
    assert got.dtype in (BF16, F32)
    half = torch.finfo(got.dtype).eps / 2
    g = _host(got)
    off, tol = np.abs(g - want), bound * (1 + half) + half * np.abs(want) + 1e-30
    assert np.isfinite(g).all(), name
    worst = np.unravel_index(np.argmax(off / tol), off.shape) if off.size else None
    assert worst is None or off[worst] <= tol[worst], (name, worst, g[worst], want[worst], off[worst] / tol[worst])


def _inputs(B, T, C, types, seed=0, state=True, rate=1.0, lead=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape = (B, T, C) if lead is None else lead
    g = -rate * torch.rand(shape, generator=gen, device="cuda") ** 3
    x = torch.randn(shape, generator=gen, device="cuda")
    s0 = torch.randn(B, C, generator=gen, device="cuda") if state else None
    return x.to(types[0]), g.to(types[1]), s0


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("B,T,C", [(1, 1, 1), (2, 3, 7), (1, 255, 64), (2, 256, 65), (1, 257, 130), (3, 1000, 96),
                                   (1, 4100, 33)])
def test_forward_and_backward(B, T, C, types):
    x, g, s0 = _inputs(B, T, C, types, seed=T + C, state=T % 2 == 1, rate=0.5)
    hx, hg, hs = _host(x), _host(g), _host(s0)
    (h, s), res = kernels.linear_recurrence_fwd(x, g, s0, out_dtype=types[2])
    want_h, want_s = ref.recurrence(hx, hg, hs)
    bound = ref.recurrence_bound(hx, hg, hs)
    assert h.dtype == types[2] and s.dtype == F32
    _near(h, want_h, bound, "h")
    _near(s, want_s, bound[:, -1], "state")
    h2, s2 = kernels.linear_recurrence(x, g, s0, out_dtype=types[2])
    assert torch.equal(h, h2) and torch.equal(s, s2)  # keeping states changes nothing
    gen = torch.Generator(device="cuda").manual_seed(7)
    gh = torch.randn(B, T, C, generator=gen, device="cuda").to(types[2])
    gs = torch.randn(B, C, generator=gen, device="cuda")
    for a, b in ((gh, gs), (gh, None), (None, gs)):
        want = ref.recurrence_bwd(hx, hg, hs, _host(a), _host(b))
        bounds = ref.recurrence_bwd_bound(hx, hg, hs, _host(a), _host(b))
        got = kernels.linear_recurrence_bwd(res, (a, b))
        assert [t.dtype for t in got] == [types[0], types[1], F32]
        for name, u, v, w in zip(("gx", "gg", "gs0"), got, want, bounds):
            _near(u, v, w, name)
    again = kernels.linear_recurrence_bwd(res, (None, gs))
    assert all(torch.equal(u, v) for u, v in zip(got, again))  # the same bits every time


@pytest.mark.parametrize("B,T,C", [(2, 1500, 64), (1, 5000, 256), (4, 700, 1000), (64, 300, 64)])
def test_long_memories_and_many_spans(B, T, C):
    """Gates near one, so that the state of the first span reaches the last."""
    for types in (TYPES[0], TYPES[3]):
        x, g, s0 = _inputs(B, T, C, types, seed=T, rate=1e-3)
        hx, hg, hs = _host(x), _host(g), _host(s0)
        (h, s), res = kernels.linear_recurrence_fwd(x, g, s0, out_dtype=types[2])
        want, _ = ref.recurrence(hx, hg, hs)
        bound = ref.recurrence_bound(hx, hg, hs)
        _near(h, want, bound, "h")
        _near(s, want[:, -1], bound[:, -1], "state")
        gh = torch.randn(B, T, C, device="cuda").to(types[2])
        got = kernels.linear_recurrence_bwd(res, (gh, None))
        for name, u, v, w in zip(("gx", "gg", "gs0"), got, ref.recurrence_bwd(hx, hg, hs, _host(gh), None),
                                 ref.recurrence_bwd_bound(hx, hg, hs, _host(gh), None)):
            _near(u, v, w, name)


def test_gates_of_every_size():
    """Closed gates (-inf: the state starts anew), tiny and growing ones."""
    B, T, C = 2, 600, 70
    x, g, s0 = _inputs(B, T, C, (F32, F32), seed=3, rate=2.0)
    g[:, ::97] = -torch.inf
    g[:, 1::13] = -60.0
    g[:, 2::7] = 0.25
    g[:, 3::11] = 0.0
    hx, hg, hs = _host(x), _host(g), _host(s0)
    (h, s), res = kernels.linear_recurrence_fwd(x, g, s0)
    fin = np.where(np.isinf(hg), -800.0, hg)  # exp(-800) is 0 in 64 bits too
    bound = ref.recurrence_bound(hx, fin, hs)
    _near(h, ref.recurrence(hx, fin, hs)[0], bound, "h")
    gh = torch.randn(B, T, C, device="cuda")
    got = kernels.linear_recurrence_bwd(res, (gh, None))
    want = ref.recurrence_bwd(hx, fin, hs, _host(gh), None)
    for name, u, v, w in zip(("gx", "gg", "gs0"), got, want, ref.recurrence_bwd_bound(hx, fin, hs, _host(gh), None)):
        _near(u, v, w, name)


def test_infinities_and_nan_stay_in_their_channel_and_after_their_token():
    B, T, C = 2, 700, 72
    x, g, s0 = _inputs(B, T, C, (BF16, BF16), seed=4)
    clean, _ = kernels.linear_recurrence(x, g, s0)
    y = x.clone()
    y[0, 300, 5], y[1, 411, 9], y[0, 20, 64] = torch.nan, torch.inf, -torch.inf
    h, s = kernels.linear_recurrence(y, g, s0)
    hit = torch.zeros(B, T, C, dtype=torch.bool, device="cuda")
    hit[0, 300:, 5] = hit[1, 411:, 9] = hit[0, 20:, 64] = True
    assert torch.equal(h[~hit], clean[~hit])
    assert not torch.isfinite(h[0, 300:, 5]).any() and not torch.isfinite(h[1, 411:, 9]).any()
    assert not torch.isfinite(s[0, 5]) and torch.isfinite(s[0, 6])
    gh = torch.randn(B, T, C, device="cuda")
    _, res = kernels.linear_recurrence_fwd(x, g, s0)
    plain = kernels.linear_recurrence_bwd(res, (gh, None))
    bad = gh.clone()
    bad[0, 400, 5] = torch.nan
    got = kernels.linear_recurrence_bwd(res, (bad, None))
    hit = torch.zeros(B, T, C, dtype=torch.bool, device="cuda")
    hit[0, :401, 5] = True
    for u, v in zip(got[:2], plain[:2]):
        assert torch.equal(u[~hit], v[~hit]) and torch.isnan(u[hit]).all()


def test_no_tokens_no_rows():
    s0 = torch.randn(2, 5, device="cuda")
    x = torch.empty(2, 0, 5, device="cuda")
    (h, s), res = kernels.linear_recurrence_fwd(x, x, s0)
    assert h.shape == (2, 0, 5) and torch.equal(s, s0)
    h, s = kernels.linear_recurrence(x, x)
    assert torch.equal(s, torch.zeros(2, 5, device="cuda"))
    gx, gg, gs0 = kernels.linear_recurrence_bwd(res, (None, s0))
    assert gx.shape == (2, 0, 5) and torch.equal(gs0, s0)
    e = torch.empty(0, 4, 5, device="cuda")
    h, s = kernels.linear_recurrence(e, e)
    assert h.shape == (0, 4, 5) and s.shape == (0, 5)


@pytest.mark.parametrize("types", [TYPES[0], TYPES[3]])
def test_views_are_read_in_place(types):
    """Halves of one projection, tokens outermost, a shifted start, an expanded batch row."""
    B, T, C = 2, 300, 37
    both = torch.randn(B, T, 2 * C + 3, device="cuda").to(types[0])
    x, g = both[..., 1:C + 1], -both[..., C + 3:].abs()
    g = torch.cat([both[..., :3], g], -1)[..., 3:]
    cases = [(x, g), (x.transpose(0, 1).contiguous().transpose(0, 1), g), (x[:1].expand(B, T, C), g),
             (x[:, 1:], g[:, :-1]), (torch.randn(C, T, B, device="cuda").to(types[0]).permute(2, 1, 0), g)]
    for a, b in cases:
        want = kernels.linear_recurrence_fwd(a.contiguous(), b.contiguous(), out_dtype=types[2])
        got = kernels.linear_recurrence_fwd(a, b, out_dtype=types[2])
        assert all(torch.equal(u, v) for u, v in zip(got[0], want[0]))
        gh = torch.randn(a.shape, device="cuda").to(types[2])
        for u, v in zip(kernels.linear_recurrence_bwd(got[1], (gh, None)),
                        kernels.linear_recurrence_bwd(want[1], (gh, None))):
            assert torch.equal(u, v)


@pytest.mark.parametrize("types", [TYPES[0], TYPES[1], TYPES[3]])
@pytest.mark.parametrize("C", [3, 64, 129])
def test_packed(C, types):
    lens = [1, 0, 300, 255, 2, 0, 513, 1, 256, 700, 0]
    cu = np.concatenate([[0], np.cumsum(lens)])
    N, n = int(cu[-1]), len(lens)
    x, g, s0 = _inputs(n, 0, C, types, seed=C, rate=0.05, lead=(N, C))
    for state in (s0, None):
        h, s = kernels.linear_recurrence_varlen(x, g, cu, state, out_dtype=types[2])
        assert h.shape == (N, C) and s.shape == (n, C)
        for i, (a, z) in enumerate(zip(cu[:-1], cu[1:])):
            first = None if state is None else _host(state[i:i + 1])
            xs, gs = _host(x[a:z])[None], _host(g[a:z])[None]
            want, end = ref.recurrence(xs, gs, first)
            bound = ref.recurrence_bound(xs, gs, first)
            _near(h[a:z][None], want, bound, ("h", i))
            if a == z:
                assert torch.equal(s[i], torch.zeros_like(s[i]) if state is None else state[i])
            else:
                _near(s[i:i + 1], end, bound[:, -1], ("state", i))
    dev = torch.from_numpy(cu).cuda()
    h2, s2 = kernels.linear_recurrence_varlen(x[None], g[None], dev, out_dtype=types[2])
    assert torch.equal(h2[0], h) and torch.equal(s2, s)
    kernels.check_varlen()


def test_packed_many_short_sequences_and_none():
    C, n = 40, 500
    lens = np.random.default_rng(0).integers(0, 7, n)
    cu = np.concatenate([[0], np.cumsum(lens)])
    x, g, s0 = _inputs(n, 0, C, (BF16, BF16), seed=9, lead=(int(cu[-1]), C))
    h, s = kernels.linear_recurrence_varlen(x, g, cu, s0)
    for i in range(n):
        a, z = cu[i], cu[i + 1]
        if a == z:
            assert torch.equal(s[i], s0[i])
            continue
        one, end = ref.recurrence(_host(x[a:z])[None], _host(g[a:z])[None], _host(s0[i:i + 1]))
        bound = ref.recurrence_bound(_host(x[a:z])[None], _host(g[a:z])[None], _host(s0[i:i + 1]))
        _near(h[a:z][None], one, bound, i)
        _near(s[i:i + 1], end, bound[:, -1], i)
    e = torch.empty(0, C, device="cuda")
    h, s = kernels.linear_recurrence_varlen(e, e, [0, 0, 0], s0[:2])
    assert h.shape == (0, C) and torch.equal(s, s0[:2])


def test_malformed_device_offsets_stay_inside():
    C, N = 16, 400
    x, g, _ = _inputs(1, 0, C, (F32, F32), seed=1, lead=(N, C))
    for cu in ([0, 500, 400], [-5, 100, 400], [0, 300, 100, 400], [10, 390], [0, 400, 900]):
        h, s = kernels.linear_recurrence_varlen(x, g, torch.tensor(cu, device="cuda"))
        assert h.shape == (N, C) and s.shape == (len(cu) - 1, C)
        with pytest.raises(kernels.KernelError):
            kernels.check_varlen()
    kernels.check_varlen()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("B,C", [(1, 1), (1, 2560), (3, 77), (256, 130)])
def test_step(B, C, types):
    x, g, s0 = _inputs(B, 0, C, types, seed=C, lead=(B, C))
    state = s0.clone()
    h = kernels.linear_recurrence_step(x, g, state, out_dtype=types[2])
    want, _ = ref.recurrence(_host(x)[:, None], _host(g)[:, None], _host(s0))
    bound = ref.recurrence_bound(_host(x)[:, None], _host(g)[:, None], _host(s0))[:, 0]
    _near(state, want[:, 0], bound, "state")
    assert torch.equal(h, state.to(types[2]))


def test_host_arrays():
    rng = np.random.default_rng(0)
    x, g, s0 = rng.normal(size=(2, 9, 5)).astype(np.float32), -rng.random((2, 9, 5)).astype(np.float32), np.ones((2, 5), np.float32)
    h, s = kernels.linear_recurrence(x, g, s0)
    assert isinstance(h, np.ndarray) and isinstance(s, np.ndarray)
    np.testing.assert_allclose(h, ref.recurrence(x, g, s0)[0], rtol=1e-5, atol=1e-5)
    t = torch.from_numpy(s0.copy())
    out = kernels.linear_recurrence_step(torch.from_numpy(x[:, 0].copy()), torch.from_numpy(g[:, 0].copy()), t)
    assert out.device.type == "cpu" and torch.equal(out, t)
    np.testing.assert_allclose(t.numpy(), ref.recurrence(x[:, :1], g[:, :1], s0)[1], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("types", [TYPES[0], TYPES[1], TYPES[3]])
def test_autograd(types):
    B, T, C = 2, 530, 65
    x, g, s0 = _inputs(B, T, C, types, seed=5, rate=0.2)
    for t in (x, g, s0):
        t.requires_grad_(True)
    h, s = kernels.linear_recurrence(x, g, s0, out_dtype=types[2])
    gh, gs = torch.randn_like(h), torch.randn_like(s)
    got = torch.autograd.grad((h, s), (x, g, s0), (gh, gs), retain_graph=True)
    assert [t.dtype for t in got] == [types[0], types[1], F32]
    want = ref.recurrence_bwd(_host(x), _host(g), _host(s0), _host(gh), _host(gs))
    for name, u, v, w in zip(("gx", "gg", "gs0"), got, want,
                             ref.recurrence_bwd_bound(_host(x), _host(g), _host(s0), _host(gh), _host(gs))):
        _near(u, v, w, name)
    # only one output used, only one input wanted
    (only,) = torch.autograd.grad(h, g, gh, retain_graph=True)
    _near(only, ref.recurrence_bwd(_host(x), _host(g), _host(s0), _host(gh), None)[1],
          ref.recurrence_bwd_bound(_host(x), _host(g), _host(s0), _host(gh), None)[1], "gg")
    (only,) = torch.autograd.grad(s, s0, gs)
    _near(only, ref.recurrence_bwd(_host(x), _host(g), _host(s0), None, _host(gs))[2],
          ref.recurrence_bwd_bound(_host(x), _host(g), _host(s0), None, _host(gs))[2], "gs0")


def test_gradients_against_differences():
    """Along a direction, differences of the kernel's own forward: second differences bound the
    truncation, the forward's bound its noise."""
    B, T, C = 1, 400, 8
    x, g, s0 = _inputs(B, T, C, (F32, F32), seed=8, rate=0.3)
    gh = torch.randn(B, T, C, device="cuda")
    _, res = kernels.linear_recurrence_fwd(x, g, s0)
    gx, gg, gs0 = kernels.linear_recurrence_bwd(res, (gh, None))
    e = 2.0**-6
    for i, grad in enumerate((gx, gg, gs0)):
        v = torch.randn_like(grad)
        side = []
        for sign in (1, 0, -1):
            args = [x, g, s0]
            args[i] = args[i] + sign * e * v
            side.append(float((gh.double() * kernels.linear_recurrence(*args)[0].double()).sum()))
        noise = float(np.sum(np.abs(_host(gh)) * 2 * ref.recurrence_bound(_host(x), _host(g), _host(s0)))) / e
        curve = abs(side[0] - 2 * side[1] + side[2]) / e
        assert abs((side[0] - side[2]) / (2 * e) - float((grad.double() * v.double()).sum())) <= noise + curve + 1e-3


def test_another_stream():
    x, g, s0 = _inputs(2, 2000, 256, (BF16, BF16), seed=6)
    want = kernels.linear_recurrence(x, g, s0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernels.linear_recurrence(x, g, s0)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(got, want))


# --- the state cache ---


@pytest.mark.parametrize("types", [TYPES[0], TYPES[3]])
def test_cache_prefill_and_decode(types):
    C, n = 96, 4
    lens = [300, 1, 520, 17]
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    cache = serving.RecurrenceStateCache(2, 9, C)
    cache.alloc(9)
    x, g, _ = _inputs(n, 0, C, types, seed=2, rate=0.1, lead=(int(cu[-1]) + 3 * n, C))
    slots = torch.tensor([7, 0, 3, 5], dtype=torch.int32, device="cuda")
    cache._pool[1] = torch.randn(10, C, device="cuda")
    before = cache._pool.clone()
    h = cache.prefill(1, slots, x[:cu[-1]], g[:cu[-1]], torch.from_numpy(cu).cuda(), out_dtype=types[2])
    plain, end = kernels.linear_recurrence_varlen(x[:cu[-1]], g[:cu[-1]], cu, before[1, slots.long()], out_dtype=types[2])
    assert torch.equal(h, plain) and torch.equal(cache.pool[1][slots.long()], end)
    rest = [i for i in range(10) if i not in slots.tolist()]
    assert torch.equal(cache._pool[1, rest], before[1, rest]) and torch.equal(cache._pool[0], before[0])
    state = end.clone()
    for t in range(3):
        xt, gt = x[int(cu[-1]) + t * n:][:n], g[int(cu[-1]) + t * n:][:n]
        out = cache.decode(1, slots, xt, gt, out_dtype=types[2])
        want = kernels.linear_recurrence_step(xt, gt, state, out_dtype=types[2])
        assert torch.equal(out, want) and torch.equal(cache.pool[1][slots.long()], state)
    # a list of slots, fixed length, int64 slots
    for s in ([7, 0, 3, 5], slots.long()):
        xs, gs = x[:n * 70].reshape(n, 70, C), g[:n * 70].reshape(n, 70, C)
        state = cache.pool[1][slots.long()].clone()
        h = cache.prefill(1, s, xs, gs)
        want, end = kernels.linear_recurrence(xs, gs, state)
        assert torch.equal(h, want) and torch.equal(cache.pool[1][slots.long()], end)
    cache.check_slots()
    saved = cache.swap_out([7, 3])
    cache.reset([7, 3])
    assert not cache.pool[:, [7, 3]].any()
    cache.swap_in([7, 3], saved)
    assert torch.equal(cache.pool[:, [7, 3]].cpu(), saved)


@pytest.mark.parametrize("types", [TYPES[0], TYPES[3]])
@pytest.mark.parametrize("T", [257, 3000, 9000])
def test_cache_prefill_in_place_over_many_spans(T, types):
    """The last span writes the row of the pool that the first has read: the same bits as a call
    with states of its own, prompts of one length and packed."""
    n, C = 3, 640
    x, g, s0 = _inputs(n, T, C, types, seed=T, rate=1e-3)
    want, end = kernels.linear_recurrence(x, g, s0, out_dtype=types[2])
    cache = serving.RecurrenceStateCache(1, 5, C)
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    for _ in range(3):
        cache.pool[0, slots.long()] = s0
        h = cache.prefill(0, slots, x, g, out_dtype=types[2])
        assert torch.equal(h, want) and torch.equal(cache.pool[0, slots.long()], end)
    cu = torch.arange(0, (n + 1) * T, T, dtype=torch.int32, device="cuda")
    flat = [t.reshape(n * T, C) for t in (x, g)]
    want, end = kernels.linear_recurrence_varlen(*flat, cu, s0, out_dtype=types[2])
    for _ in range(3):
        cache.pool[0, slots.long()] = s0
        h = cache.prefill(0, slots, *flat, cu, out_dtype=types[2])
        assert torch.equal(h, want) and torch.equal(cache.pool[0, slots.long()], end)


def test_cache_padding_and_bad_slots():
    C = 70
    cache = serving.RecurrenceStateCache(1, 4, C)
    cache._pool[:] = torch.randn(1, 5, C, device="cuda")
    before = cache._pool.clone()
    x, g, _ = _inputs(4, 0, C, (BF16, BF16), seed=1, lead=(4, C))
    slots = torch.tensor([2, -1, 4, 0], dtype=torch.int32, device="cuda")
    out = torch.full((4, C), 7.0, dtype=BF16, device="cuda")
    assert cache.decode(0, slots, x, g, out) is out
    assert not out[1:3].any() and out[[0, 3]].any(1).all()
    assert torch.equal(cache._pool[0, [1, 3, 4]], before[0, [1, 3, 4]])
    cache.check_slots()  # padding of a decode batch is no error
    now = cache._pool.clone()
    xs, gs = x[:, None].expand(4, 300, C), g[:, None].expand(4, 300, C)
    h = cache.prefill(0, slots, xs, gs)
    zero, _ = kernels.linear_recurrence(xs[1:3], gs[1:3])
    assert torch.equal(h[1:3], zero)  # from a zero state
    assert torch.equal(cache._pool[0, [1, 3, 4]], now[0, [1, 3, 4]])
    with pytest.raises(ValueError):
        cache.check_slots()
    cache.check_slots()
    far = torch.tensor([2, 2**32 + 1, -(2**32), 0], device="cuda")  # not slot 1 and 0
    now = cache._pool.clone()
    cache.prefill(0, far, xs, gs)
    assert torch.equal(cache._pool[0, [1, 3, 4]], now[0, [1, 3, 4]])
    with pytest.raises(ValueError):
        cache.check_slots()


def test_graph_replays():
    """Prefill and decode captured, replayed with eager work between the replays."""
    C, n, N = 128, 3, 900
    x, g, _ = _inputs(n, 0, C, (BF16, BF16), seed=2, rate=0.1, lead=(N, C))
    cu = torch.tensor([0, 500, 501, N], dtype=torch.int32, device="cuda")
    slots = torch.tensor([1, 4, 2], dtype=torch.int32, device="cuda")
    cache, eager = serving.RecurrenceStateCache(1, 6, C), serving.RecurrenceStateCache(1, 6, C)
    kernels.check_varlen()

    def work(c):
        h = c.prefill(0, slots, x, g, cu, out_dtype=BF16)
        return h, c.decode(0, slots, x[:n], g[:n])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(cache)
    torch.cuda.current_stream().wait_stream(side)
    work(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(cache)
    for i in range(4):
        x.copy_(torch.randn(N, C, device="cuda"))
        slots.copy_(torch.tensor([[1, 4, 2], [0, 5, 3]][i % 2], dtype=torch.int32))
        want = work(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(outs, want))
        assert torch.equal(cache.pool, eager.pool)
