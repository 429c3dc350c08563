"""The bounds of ``decay_accuracy`` see a lost part of a factor: the chunked form in 64 bits with its
factors cut to bf16 parts stays inside them with the parts that the kernels keep, and not with one less."""

from __future__ import annotations

import pytest
import torch

from oracle import decay_oracle as ref
from tests import decay_accuracy as acc

SHAPES = [(2, 130, 4, 2, 64), (1, 200, 2, 2, 128), (1, 150, 2, 1, 80)]


@pytest.mark.parametrize("B,T,Hq,H,D", SHAPES)
def test_the_chunked_form_is_the_same(B, T, Hq, H, D):
    x = acc.inputs(B, T, Hq, H, D, acc.F32)[:5]
    for got, want in zip(ref.chunked(*x, scale=0.7), ref.decay(*x, 0.7)):
        assert torch.allclose(got, want, rtol=1e-10, atol=1e-12)


@pytest.mark.parametrize("B,T,Hq,H,D", SHAPES)
def test_parts_of_bf16_inputs_products(B, T, Hq, H, D):
    x = acc.inputs(B, T, Hq, H, D, acc.BF16)[:5]
    want, spread = ref.decay(*x, 0.7), ref.spread(*x, 0.7)
    eps = acc.of_factors(acc.BF16, T, Hq // H, D), acc.of_sums(T, 1, D)

    def off(i, **parts):
        return ref.rms(ref.chunked(*x, 0.7, **parts)[i] - want[i])

    for out in (acc.F32, acc.BF16):
        o = ref.chunked(*x, 0.7, factors=2)[0].to(out)
        acc.check(o, want[0], spread[0], eps[0])
        with pytest.raises(AssertionError):
            acc.check(ref.chunked(*x, 0.7, factors=1)[0].to(out), want[0], spread[0], eps[0])
    assert off(1, decayed=3) <= acc.bound(want[1], spread[1], acc.F32, eps[1]) < off(1, decayed=2)


@pytest.mark.parametrize("B,T,Hq,H,D", SHAPES)
def test_parts_of_fp32_inputs(B, T, Hq, H, D):
    x = acc.inputs(B, T, Hq, H, D, acc.F32)[:5]
    want, spread = ref.decay(*x, 0.7), ref.spread(*x, 0.7)
    for i, eps in enumerate((acc.of_factors(acc.F32, T, Hq // H, D), acc.of_sums(T, 1, D))):
        most = acc.bound(want[i], spread[i], acc.F32, eps)
        three = ref.chunked(*x, 0.7, chunk=32, inputs=3, factors=3, decayed=3)[i]
        assert ref.rms(three - want[i]) <= most < ref.rms(ref.chunked(*x, 0.7, inputs=2)[i] - want[i])
    o = ref.chunked(*x, 0.7, factors=2)[0] - want[0]
    assert acc.bound(want[0], spread[0], acc.F32, acc.of_factors(acc.F32, T, Hq // H, D)) < ref.rms(o)


def test_spreads_are_of_the_terms():
    """One sum over pairs of tokens, written out."""
    q, k, v, g, s0, go, gs = acc.inputs(1, 5, 1, 1, 3, acc.F32)
    _, state = ref.spread(q, k, v, g, s0)
    G = torch.cumsum(g[0, :, 0].double(), 0)
    terms = [torch.exp(G[-1]) * s0[0, 0].double()]
    terms += [torch.exp(G[-1] - G[t]) * k[0, t, 0, :, None].double() * v[0, t, 0].double() for t in range(5)]
    assert torch.allclose(state[0, 0], sum(t**2 for t in terms).sqrt())
    gv = ref.spread_bwd(q, k, v, g, s0, go, gs)[2]
    last = ((gs[0, 0].double() * k[0, 4, 0, :, None].double())**2).sum(0)
    last += ((q[0, 4, 0, :, None].double() * go[0, 4, 0].double() * k[0, 4, 0, :, None].double())**2).sum(0)
    assert torch.allclose(gv[0, 4, 0], last.sqrt())


@pytest.mark.parametrize("dtype", [acc.BF16, acc.F32])
def test_what_spans_hand_on_is_seen(dtype):
    """Slow decays: a span that does not start from the state before it, or whose gradients miss what comes
    from before it, is far outside of the bounds."""
    T, at = 1100, 576
    x = acc.slow(1, T, 2, 1, 16, dtype)
    q, k, v, g, s0, go, gs = x
    want, spread = ref.decay(q, k, v, g, s0), ref.spread(q, k, v, g, s0)
    lost = [t[:, at:] for t in (q, k, v, g)]
    o, s = ref.decay(*lost)
    for got, e, m, eps in ((o, want[0][:, at:], spread[0][:, at:], acc.of_factors(dtype, T, 2, 16)),
                           (s, want[1], spread[1], acc.of_sums(T, 1, 16))):
        assert ref.rms(got - e) > 1000 * acc.bound(e, m, acc.F32, eps)
    grads, sizes = ref.decay_bwd(*x[:5], go, gs), ref.spread_bwd(*x)
    got = ref.decay_bwd(*lost, None, go[:, at:], gs)
    most = acc.bound(grads[0][:, at:], sizes[0][:, at:], acc.F32, acc.of_factors(dtype, T, 2, 16))
    assert ref.rms(got[0] - grads[0][:, at:]) > 100 * most
    assert ref.rms(got[3] - grads[3][:, at:]) > 100 * acc.bound_gates(sizes[3], T, 2, 16)


def test_a_lost_part_of_the_decays_gradient_is_seen():
    """The state as one bf16 part in what sums into it (dL/dg_t = <gradient of the state, e^g state before>)."""
    B, T, Hq, H, D = 1, 200, 2, 2, 64
    x = acc.inputs(B, T, Hq, H, D, acc.BF16)
    want, spread = ref.decay_bwd(*x)[3], ref.spread_bwd(*x)[3]
    most = acc.bound_gates(spread, T, 1, D)
    q, k, v, g, s0, go, gs = x
    # a token's r: q_t . (e^{G} S go_t) from the state at its chunk's start, with that state in parts
    off = {}
    for parts in (1, 2):
        total = 0.0
        for a in range(64, T, 64):
            z = min(a + 64, T)
            state = ref.decay(q[:, :a], k[:, :a], v[:, :a], g[:, :a], s0)[1]
            G = torch.exp(torch.cumsum(g[:, a:z].double(), 1))
            r = G * torch.einsum("bthd,bhde,bthe->bth", q[:, a:z].double(), ref.planes(state, parts) - state,
                                 go[:, a:z].double())
            total += r.square().sum().item()  # (an error of the gradient at each token that r is summed to)
        off[parts] = (total / want.numel()) ** 0.5
    assert off[2] < most < off[1]
