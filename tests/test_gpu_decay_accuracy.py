"""Decay attention on the GPU against the 64-bit form, by the root mean square of what it is off by: the
bounds (``decay_accuracy``) see a bf16 part of a factor that is lost, which the largest errors of
``test_gpu_decay_attention.py`` do not."""

from __future__ import annotations

import pytest
import torch

from oracle import decay_oracle as ref
from prometheus_amd import kernels, serving
from tests import decay_accuracy as acc

pytestmark = pytest.mark.gpu
BF16, F32 = acc.BF16, acc.F32

SHAPES = [(2, 130, 4, 2, 64), (1, 200, 2, 2, 128), (1, 150, 2, 1, 80), (1, 130, 1, 1, 256)]


def gpu(*xs):
    return [None if x is None else x.cuda() for x in xs]


@pytest.mark.parametrize("B,T,Hq,H,D", SHAPES)
@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (BF16, F32), (F32, F32)])
def test_outputs(B, T, Hq, H, D, dtype, out):
    x = acc.inputs(B, T, Hq, H, D, dtype, seed=T)[:5]
    o, s = kernels.decay_attention(*gpu(*x), scale=0.7, out_dtype=out)
    want, spread = ref.decay(*x, 0.7), ref.spread(*x, 0.7)
    acc.check(o, want[0], spread[0], acc.of_factors(dtype, T, Hq // H, D))
    acc.check(s, want[1], spread[1], acc.of_sums(T, 1, D))


@pytest.mark.parametrize("B,T,Hq,H,D", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradients_of_the_inputs(B, T, Hq, H, D, dtype):
    q, k, v, g, s0, go, gs = acc.inputs(B, T, Hq, H, D, dtype, seed=T)
    _, res = kernels.decay_attention_fwd(*gpu(q, k, v, g, s0), scale=0.7)
    got = kernels.decay_attention_bwd(res, gpu(go, gs))
    want, spread = ref.decay_bwd(q, k, v, g, s0, go, gs, 0.7), ref.spread_bwd(q, k, v, g, s0, go, gs, 0.7)
    for i in range(3):
        assert got[i].dtype == dtype
        acc.check(got[i], want[i], spread[i], acc.of_factors(dtype, T, Hq // H, D))


@pytest.mark.parametrize("B,T,Hq,H,D", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("gates", [True, False])
def test_gradient_of_the_first_state(B, T, Hq, H, D, dtype, gates):
    """As near whether the decays' gradient is taken with it or not."""
    q, k, v, g, s0, go, gs = acc.inputs(B, T, Hq, H, D, dtype, seed=T)
    dev = gpu(q, k, v, g, s0)
    for x in (dev if gates else dev[:3] + dev[4:]):
        x.requires_grad_(True)
    o, s = kernels.decay_attention(*dev, scale=0.7)
    (got,) = torch.autograd.grad((o, s), dev[4], gpu(go, gs))
    want, spread = ref.decay_bwd(q, k, v, g, s0, go, gs, 0.7), ref.spread_bwd(q, k, v, g, s0, go, gs, 0.7)
    acc.check(got, want[4], spread[4], acc.of_sums(T, Hq // H, D))


@pytest.mark.parametrize("B,T,Hq,H,D", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradient_of_the_decays(B, T, Hq, H, D, dtype):
    x = acc.inputs(B, T, Hq, H, D, dtype, seed=T)
    _, res = kernels.decay_attention_fwd(*gpu(*x[:5]), scale=0.7)
    gg = kernels.decay_attention_bwd(res, gpu(*x[5:]))[3]
    want, spread = ref.decay_bwd(*x, 0.7)[3], ref.spread_bwd(*x, 0.7)[3]
    acc.check_gates(gg, want, spread, T, Hq // H, D)


@pytest.mark.parametrize("B,T,Hq,H,D", [(1, 1100, 4, 2, 64), (2, 1300, 2, 1, 128), (1, 900, 2, 2, 33)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_slow_decays_through_many_spans(B, T, Hq, H, D, dtype):
    """States that live through the whole sequence, from a state and with a gradient of the last one."""
    x = acc.slow(B, T, Hq, H, D, dtype)
    (o, s), res = kernels.decay_attention_fwd(*gpu(*x[:5]), scale=0.7)
    got = kernels.decay_attention_bwd(res, gpu(*x[5:]))
    want, spread = ref.decay(*x[:5], 0.7), ref.spread(*x[:5], 0.7)
    acc.check(o, want[0], spread[0], acc.of_factors(dtype, T, Hq // H, D))
    acc.check(s, want[1], spread[1], acc.of_sums(T, 1, D))
    want, spread = ref.decay_bwd(*x, 0.7), ref.spread_bwd(*x, 0.7)
    for i in range(3):
        acc.check(got[i], want[i], spread[i], acc.of_factors(dtype, T, Hq // H, D))
    acc.check_gates(got[3], want[3], spread[3], T, Hq // H, D)
    acc.check(got[4], want[4], spread[4], acc.of_sums(T, Hq // H, D))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Hq,H", [(2, 2), (4, 2)])
def test_slow_decays_of_packed_prompts_in_slots(dtype, Hq, H):
    """Sequences of several spans each, into a cache's slots and on from there."""
    D, lengths = 64, [1500, 0, 700, 3]
    q, k, v, g, *_ = acc.slow(1, sum(lengths), Hq, H, D, dtype)
    cache = serving.DecayStateCache(1, 6, H, D)
    s0 = torch.randn(4, H, D, D, generator=torch.Generator().manual_seed(1))
    slots = torch.tensor([3, 5, 0, 2], device="cuda")
    cache.pool[0, slots] = s0.cuda()
    cu = torch.tensor([0, *lengths]).cumsum(0).cuda()
    o = cache.prefill(0, slots, *gpu(q, k, v, g), cu)
    cache.check_slots()
    kernels.check_varlen()
    a = 0
    for i, n in enumerate(lengths):
        part = [t[:, a:a + n] for t in (q, k, v, g)]
        want, spread = ref.decay(*part, s0[i:i + 1]), ref.spread(*part, s0[i:i + 1])
        if n:
            acc.check(o[:, a:a + n], want[0], spread[0], acc.of_factors(dtype, n, Hq // H, D))
        acc.check(cache.pool[0, slots[i]][None], want[1], spread[1], acc.of_sums(n, 1, D))
        a += n


@pytest.mark.parametrize("H,D,T", [(300, 24, 700), (60, 130, 500)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_heads_in_spans(H, D, T, dtype):
    """Where the card holds just twice as many workgroups as there are heads."""
    x = acc.slow(1, T, H, H, D, dtype)
    o, s = kernels.decay_attention(*gpu(*x[:5]))
    some = [0, H // 2, H - 1]
    part = [t[:, :, some] for t in x[:4]]
    want, spread = ref.decay(*part, x[4][:, some]), ref.spread(*part, x[4][:, some])
    acc.check(o[:, :, some], want[0], spread[0], acc.of_factors(dtype, T, 1, D))
    acc.check(s[:, some], want[1], spread[1], acc.of_sums(T, 1, D))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,D", [(20, 33), (100, 16), (150, 64), (130, 128), (90, 200)])
def test_whole_numbers_come_out_whole(T, D, dtype):
    """One-hot rows of whole numbers, no decay, a first state of whole numbers up to 2^19, more than two bf16
    parts hold (17 bits), gradients from 16 tokens: every sum stays below 2^24, so that the decays' gradient, the
    states and their gradient are exact in fp32 if no factor has lost a part."""
    gen = torch.Generator().manual_seed(T)

    def one_hot(most):
        x = torch.zeros(1, T, 2, D)
        return x.scatter_(3, torch.randint(D, (1, T, 2, 1), generator=gen),
                          torch.randint(1, most + 1, (1, T, 2, 1), generator=gen).float()).to(dtype)

    q, k, v, go = one_hot(1), one_hot(1), one_hot(3), one_hot(1)
    go *= (torch.randperm(T, generator=gen) < 16)[None, :, None, None]
    s0 = torch.randint(-(2**19), 2**19 + 1, (1, 2, D, D), generator=gen).float()
    g = torch.zeros(1, T, 2)
    (_, s), res = kernels.decay_attention_fwd(*gpu(q, k, v, g, s0))
    got = kernels.decay_attention_bwd(res, (go.cuda(), None))
    assert torch.equal(s.cpu().double(), ref.decay(q, k, v, g, s0)[1])
    want = ref.decay_bwd(q, k, v, g, s0, go, None)
    assert want[3].abs().max() < 2**24
    assert torch.equal(got[3].cpu().double(), want[3]) and torch.equal(got[4].cpu().double(), want[4])
