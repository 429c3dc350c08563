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


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,D", [(100000, 16), (70000, 128), (200, 64)])
def test_other_values_keep_their_bits(dtype, T, D):
    """Groups of query heads, one after another in a workgroup where there is work enough: a NaN in v changes
    its own column from its token on, one in k its group's gq from there on, one in q its key head's gk up to
    there, and no other bit."""
    Hq, H, token, column = 4, 2, T // 2 + 5, 9
    gen = torch.Generator(device="cuda").manual_seed(T)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    q, k, v = normal(1, T, Hq, D).to(dtype), (normal(1, T, H, D) / D**0.5).to(dtype), normal(1, T, H, D).to(dtype)
    g, s0, go = -0.3 * torch.rand(1, T, H, generator=gen, device="cuda"), normal(1, H, D, D), normal(1, T, Hq, D).to(dtype)

    def run(q, k, v):
        (o, s), res = kernels.decay_attention_fwd(q, k, v, g, s0)
        gq, gk, gv, _, _ = kernels.decay_attention_bwd(res, (go, None))
        return {"o": o, "s": s, "gq": gq, "gk": gk, "gv": gv}

    def with_nan(x, head):
        x = x.clone()
        x[0, token, head, column] = NAN
        return x

    def same(name, got, open_values):
        """The same bits, but for the values of ``open_values``, which are not finite."""
        want = clean[name].clone()
        assert not got[name][open_values].isfinite().any(), name
        want[open_values] = got[name][open_values] = 0.0
        assert torch.equal(got[name], want), name

    def mask(name, *index):
        m = torch.zeros_like(clean[name], dtype=torch.bool)
        m[(0, *index)] = True
        return m

    clean = run(q, k, v)
    later, earlier, whole = slice(token, T), slice(0, token + 1), slice(None)
    got = run(q, k, with_nan(v, 1))
    same("o", got, mask("o", later, slice(2, 4), column))
    same("s", got, mask("s", 1, whole, column))
    same("gv", got, mask("gv", slice(0, 0)))
    same("gk", got, mask("gk", slice(token, token + 1), 1))
    got = run(q, with_nan(k, 1), v)
    same("gq", got, mask("gq", later, slice(2, 4), column))
    got = run(with_nan(q, 3), k, v)
    same("gk", got, mask("gk", earlier, 1, column))
    same("gq", got, mask("gq", slice(0, 0)))
