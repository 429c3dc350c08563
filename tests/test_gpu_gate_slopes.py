"""Gradients of the gated norm's gate where the gate is nearly closed or wide open."""

from __future__ import annotations

import pytest
import torch

from oracle import decay_oracle as ref
from prometheus_amd import kernels

pytestmark = pytest.mark.gpu


def slope(z, activation):
    """s (1 - s), or s + z s (1 - s). (Not by autograd: its 1 - s has lost three digits at z = 30 in 64 bits.)"""
    e = torch.exp(-z.abs())
    s, d = torch.where(z < 0, e, 1.0) / (1 + e), e / (1 + e)**2
    return s + z * d if activation == "silu" else d


def test_the_slopes_against_autograd():
    z = torch.linspace(-8.0, 8.0, 101, dtype=torch.float64, requires_grad=True)
    for activation, f in (("silu", torch.nn.functional.silu), ("sigmoid", torch.sigmoid)):
        (g,) = torch.autograd.grad(f(z).sum(), z)
        assert torch.allclose(g, slope(z.detach(), activation), rtol=1e-11, atol=1e-14)


@pytest.mark.parametrize("activation", ["silu", "sigmoid"])
@pytest.mark.parametrize("C", [33, 128, 2000])
def test_slopes_of_closed_and_open_gates(activation, C):
    """fp32: e^-|z| is off by |z| 2^-24 twice, where its exponent is rounded and for the constant in it; the
    exponential, the reciprocal, the norm's root and quotient by 2^-23 each, every product and sum by 2^-24:
    8, 8 of a lane's and 10 from lane to lane, of which the root takes half. Under 40 in all, and nothing is
    lost to a difference, but for silu's slope near its own zero."""
    gen = torch.Generator().manual_seed(C)
    x, gy = (torch.randn(6, C, generator=gen) for _ in range(2))
    z = torch.linspace(-30.0, 30.0, 6 * C).view(6, C)[:, torch.randperm(C, generator=gen)]
    if activation == "silu":
        z = torch.where((z + 1.2785).abs() < 0.5, 2.0, z)
    want = gy.double() * ref.gated(x, torch.full_like(z, 100.0), activation="sigmoid") * slope(z.double(), activation)
    y, res = kernels.gated_norm_fwd(x.cuda(), z.cuda(), activation=activation)
    got = kernels.gated_norm_bwd(res, gy.cuda())[1].cpu().double()
    off = (got - want).abs()
    # (silu's slope s + z s (1 - s) is at least a tenth of its terms outside of the range taken out)
    allowed = (2 * z.abs().double() + 40) * 2.0**-24 * want.abs() * (10 if activation == "silu" else 1)
    assert bool((off <= allowed).all()), (off / allowed).max().item()
