"""Infinities and NaN in decay attention's inputs reach the outputs that they reach token by token, and no
other: nothing of a token comes out at the tokens before it (or, in a gradient, behind it)."""

from __future__ import annotations

import pytest
import torch

from oracle import decay_oracle as ref
from prometheus_amd import kernels
from tests import decay_accuracy as acc

pytestmark = pytest.mark.gpu
BF16, F32 = acc.BF16, acc.F32
INF, NAN = float("inf"), float("nan")

SHAPES = [(2, 150, 2, 2, 64), (1, 150, 4, 2, 128), (1, 150, 1, 1, 200), (1, 70, 2, 1, 33), (1, 1200, 2, 1, 64)]


def gpu(*xs):
    return [None if x is None else x.cuda() for x in xs]


def check(got, want, spread, eps):
    """The same values are finite, and those are near."""
    got = got.detach().cpu()
    assert torch.equal(got.isfinite(), want.isfinite())
    there = want.isfinite()
    acc.check(got[there], want[there], spread[there], eps)


def clean(x):
    return torch.nan_to_num(x, 0.0, 0.0, 0.0)


@pytest.mark.parametrize("B,T,Hq,H,D", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("token,column,value", [(0, 0, NAN), (5, 17, INF), (16, 3, -INF), (31, 32, NAN), (40, 7, NAN),
                                                (63, 31, INF), (64, 0, NAN)])
def test_values(B, T, Hq, H, D, dtype, token, column, value):
    q, k, v, g, s0, *_ = acc.inputs(B, T, Hq, H, D, dtype, seed=T)
    v[0, token, -1, column] = value
    if D > 64:
        v[0, token + 3, -1, 60] = NAN  # another column, of a later token
    o, s = kernels.decay_attention(*gpu(q, k, v, g, s0))
    want = ref.decay(q, k, v, g, s0)
    spread = [x.nan_to_num(0.0, 0.0, 0.0) for x in ref.spread(q, k, clean(v), g, s0)]
    check(o, want[0], spread[0], acc.of_factors(dtype, T, Hq // H, D) + 2.0**-24 * T)
    check(s, want[1], spread[1], acc.of_sums(T, 1, D))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("which", ["q", "k", "g"])
def test_queries_keys_and_decays(dtype, which):
    q, k, v, g, s0, *_ = acc.inputs(1, 100, 2, 2, 64, dtype)
    {"q": q, "k": k, "g": g}[which][0, 37, 1] = NAN
    o, s = kernels.decay_attention(*gpu(q, k, v, g, s0))
    for got, want in zip((o, s), ref.decay(q, k, v, g, s0)):
        assert torch.equal(got.cpu().isfinite(), want.isfinite())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Hq,H", [(2, 2), (4, 2)])
@pytest.mark.parametrize("T", [100, 1200])
def test_what_stands_behind_the_valid_tokens(dtype, Hq, H, T):
    """A padded row: rubbish in k and v behind its tokens, no gradient from there."""
    n, D = T - 23, 64
    q, k, v, g, s0, go, _ = acc.inputs(2, T, Hq, H, D, dtype)
    go[0, n:] = 0.0
    k[0, n:], v[0, n:] = NAN, INF
    x = gpu(q, k, v, g, s0)
    (o, _), res = kernels.decay_attention_fwd(*x)
    *grads, gg, _ = kernels.decay_attention_bwd(res, (go.cuda(), None))
    got = [o, *grads]
    short = [t[:, :n] for t in (q, k, v, g)]
    want = [ref.decay(*short, s0)[0], *ref.decay_bwd(*short, s0, go[:, :n], None)[:3]]
    spread = [ref.spread(*short, s0)[0], *ref.spread_bwd(*short, s0, go[:, :n], None)[:3]]
    for a, b, c in zip(got, want, spread):
        assert a[0, :n].isfinite().all()
        acc.check(a[:1, :n], b[:1], c[:1], acc.of_factors(dtype, T, Hq // H, D))
    assert gg[0, :n].isfinite().all()
    # (the second row is whole)
    assert all(a[1].isfinite().all() for a in (*got, gg))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("token", [0, 20, 63, 64, 99])
def test_gradients(dtype, token):
    """k reaches later tokens' gq, q and go earlier tokens' gk and gv."""
    for which in range(3):
        q, k, v, g, s0, go, gs = acc.inputs(1, 100, 2, 2, 64, dtype)
        (q, k, go)[which][0, token, 0, 5] = NAN
        _, res = kernels.decay_attention_fwd(*gpu(q, k, v, g, s0))
        got = kernels.decay_attention_bwd(res, gpu(go, gs))
        want = ref.decay_bwd(q, k, v, g, s0, go, gs)
        for i in (0, 1, 2, 4):
            assert torch.equal(got[i].cpu().isfinite(), want[i].isfinite()), (which, i)
