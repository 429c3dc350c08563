"""Decay attention and the norms around it on the GPU at the edges of their sizes."""

from __future__ import annotations

import math

import pytest
import torch

from prometheus_amd import kernels

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
