"""Decay attention on the GPU against the 64-bit form, by the root mean square of what it is off by: the
bounds (``decay_accuracy``) see a bf16 part of a factor that is lost, which the largest errors of
``test_gpu_decay_attention.py`` do not."""

from __future__ import annotations

import pytest
import torch

from oracle import decay_oracle as ref
from prometheus_amd import kernels
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
