"""Decay attention and the norms around it on the GPU at the edges of their sizes."""

from __future__ import annotations

import math

import pytest
import torch

from prometheus_amd import kernels
from tests.test_decay_limits_cpu import EMPTY

pytestmark = pytest.mark.gpu
MOST = 2**31 - 1 - 1024  # tokens of a sequence


@pytest.mark.parametrize("cu", [None, [0, MOST], [0, 1 << 20, MOST]])
def test_as_many_tokens_as_a_call_takes(cu):
    """The state halves and gains one at each token: it is 2 - 2^-t after t more, in every span."""
    x = torch.ones(1, 1, 1, 1, dtype=torch.bfloat16, device="cuda").expand(1, MOST, 1, 1)
    g = torch.full((1,), -math.log(2.0), device="cuda")
    if cu is None:
        o, s = kernels.decay_attention(x, x, x, g)
    else:
        o, s = kernels.decay_attention_varlen(x, x, x, g, cu)
    o = o.flatten()
    for a in (cu or [0])[:-1] or [0]:
        want = [2.0 - 2.0**-t for t in range(8)]
        assert o[a:a + 8].tolist() == want and bool((o[a + 8:a + 64] >= want[-1]).all())
        o[a:a + 64] = 2.0
    low, high = o.aminmax()
    assert low.item() == high.item() == 2.0
    assert (s - 2.0).abs().max().item() < 1e-5


@pytest.mark.parametrize("shape", EMPTY)
@pytest.mark.parametrize("kind", ["gpu", "view", "fp16", "cpu", "numpy"])
def test_norms_of_no_rows(shape, kind):
    """Both directions, through autograd and without, where the fast path of contiguous tensors is not taken."""
    x, w = torch.zeros(shape), torch.ones(shape[-1])
    if kind != "cpu" and kind != "numpy":
        x, w = x.cuda(), w.cuda()
    if kind == "view":
        x = torch.zeros(*shape[:-1], shape[-1] + 3, device="cuda")[..., 1:shape[-1] + 1]
    if kind == "fp16":
        x = x.half()
    if kind == "numpy":
        x, w = x.numpy(), w.numpy()
    y, res = kernels.gated_norm_fwd(x, x, w)
    gx, gz, gw = kernels.gated_norm_bwd(res, y)
    assert y.shape == gx.shape == gz.shape == shape and gw.shape == w.shape and not gw.any()
    (y, h), res = kernels.residual_norm_fwd(x, x, w, post_weight=w)
    gx, gr, gw, gwp = kernels.residual_norm_bwd(res, (y, h))
    assert y.shape == h.shape == gx.shape == gr.shape == shape and not gw.any() and not gwp.any()
    if kind != "numpy":
        leaves = [x.clone().requires_grad_(True), x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        for f in (kernels.gated_norm, lambda *a: kernels.residual_norm(*a)[0]):
            grads = torch.autograd.grad(f(*leaves).sum(), leaves)
            assert grads[0].shape == shape and not grads[2].any()


def test_gradients_of_as_many_tokens_as_a_call_takes():
    """The same from both ends: gq is 2 - 2^-t after t more tokens, gk and gv before as many, and every token
    adds the decayed state before it times the gradient behind it, 2 of them, to the one decay's gradient."""
    x = torch.ones(1, 1, 1, 1, dtype=torch.bfloat16, device="cuda").expand(1, MOST, 1, 1)
    g = torch.full((1,), -math.log(2.0), device="cuda")
    _, res = kernels.decay_attention_fwd(x, x, x, g)
    gq, gk, gv, gg, gs = kernels.decay_attention_bwd(res, (x, None))
    want = [2.0 - 2.0**-t for t in range(8)]
    for grad, ends in ((gq, slice(0, 64)), (gk, slice(MOST - 64, MOST)), (gv, slice(MOST - 64, MOST))):
        grad = grad.flatten()
        part = grad[ends] if ends.start == 0 else grad[ends].flip(0)
        assert part[:8].tolist() == want and bool((part[8:] >= want[-1]).all())
        grad[ends] = 2.0
        low, high = grad.aminmax()
        assert low.item() == high.item() == 2.0
    assert gg.item() == pytest.approx(2.0 * MOST, rel=1e-6)
    assert gs.item() == pytest.approx(1.0, rel=1e-6)
