"""Decay attention and the norms around it as a decoder uses them: two blocks trained, against the same
in 64 bits, and served from the state cache, against the whole sequences.

fp32: every operator's own error is at most (T + 64) 2^-23 of its terms (T 70), every product of C = 128
terms at most 128 2^-23; two blocks of about ten such steps each, whose norms keep every value of order
one: 20 * 134 * 2^-23 = 3.2e-4 relative to the largest value, in gradients twice that.
"""

from __future__ import annotations

import pytest
import torch

from oracle import decay_oracle as ref
from prometheus_amd import kernels, serving

pytestmark = pytest.mark.gpu
HQ, H, D, WIDTH, T = 4, 2, 32, 128, 70


def weights(seed):
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape, scale):
        return torch.randn(shape, generator=gen) * scale

    return {"inner": normal(WIDTH, (2 * HQ + 2 * H) * D + H, scale=WIDTH**-0.5), "heads": 1 + normal(D, scale=0.1),
            "outer": normal(HQ * D, WIDTH, scale=(HQ * D)**-0.5), "post": 1 + normal(WIDTH, scale=0.1),
            "pre": 1 + normal(WIDTH, scale=0.1)}


def parts(y, w):
    """q, k, v, z and log-decays of one projection."""
    p = y @ w["inner"]
    q, k, v, z, g = p.split([HQ * D, H * D, H * D, HQ * D, H], -1)
    return *(x.unflatten(-1, (-1, D)) for x in (q, k, v, z)), -torch.nn.functional.softplus(g)


def block(y, h, w, attend):
    q, k, v, z, g = parts(y, w)
    o = kernels.gated_norm(attend(q, k, v, g), z, w["heads"])
    return kernels.residual_norm(o.flatten(-2) @ w["outer"], h, w["pre"], post_weight=w["post"], scale=0.5)


def plain(x, ws):
    """The same in 64 bits, differentiable."""
    y, h = x, x
    for w in ws:
        q, k, v, z, g = parts(y, w)
        s = torch.zeros(x.shape[0], H, D, D, dtype=torch.float64)
        out = []
        for t in range(x.shape[1]):
            s = torch.exp(g[:, t])[..., None, None] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
            out.append((q[:, t].unflatten(1, (H, -1)).unsqueeze(-2) @ s.unsqueeze(2)).squeeze(-2).flatten(1, 2) * D**-0.5)
        o = ref.gated(torch.stack(out, 1), z, w["heads"])
        y, h = ref.residual(o.flatten(-2) @ w["outer"], h, w["pre"], w["post"], 0.5)
    return y, h


def close(got, want, tol):
    assert (got.detach().cpu().double() - want).abs().max() <= tol * want.abs().max()


def test_trained():
    ws = [weights(i) for i in range(2)]
    x = torch.randn(2, T, WIDTH, generator=torch.Generator().manual_seed(9))
    dev = [{n: t.cuda().requires_grad_(True) for n, t in w.items()} for w in ws]
    y = h = xd = x.cuda().requires_grad_(True)
    for w in dev:
        y, h = block(y, h, w, lambda *a: kernels.decay_attention(*a, scale=D**-0.5)[0])
    leaves = [xd, *(t for w in dev for t in w.values())]
    got = torch.autograd.grad(y.square().mean() + h.square().mean(), leaves)
    exact = [{n: t.double().requires_grad_(True) for n, t in w.items()} for w in ws]
    xe = x.double().requires_grad_(True)
    ye, he = plain(xe, exact)
    close(y, ye.detach(), 3.2e-4)
    close(h, he.detach(), 3.2e-4)
    want = torch.autograd.grad(ye.square().mean() + he.square().mean(), [xe, *(t for w in exact for t in w.values())])
    for a, b in zip(got, want):
        close(a, b, 6.4e-4)


@torch.no_grad()
def test_served():
    ws = [{n: t.cuda() for n, t in weights(i).items()} for i in range(2)]
    lengths, more = [40, 1, 25], 4
    xs = [torch.randn(1, n + more, WIDTH, generator=torch.Generator().manual_seed(n)).cuda() for n in lengths]
    cache = serving.DecayStateCache(2, 5, H, D)
    slots = torch.tensor(cache.alloc(3)[::-1], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, *lengths]).cumsum(0).int().cuda()

    def run(x, attend):
        y = h = x
        for layer, w in enumerate(ws):
            y, h = block(y, h, w, lambda *a: attend(layer, *a))
        return y

    packed = torch.cat([x[0, :n] for x, n in zip(xs, lengths)])
    got = [[p] for p in run(packed, lambda i, *a: cache.prefill(i, slots, *a, cu, scale=D**-0.5)).split(lengths)]
    for t in range(more):
        now = torch.cat([x[0, n + t:n + t + 1] for x, n in zip(xs, lengths)])
        y = run(now, lambda i, *a: cache.decode(i, slots, *(u.contiguous() for u in a), scale=D**-0.5))
        for i in range(3):
            got[i].append(y[i:i + 1])
    cache.check_slots()
    kernels.check_varlen()
    for parts_, x in zip(got, xs):
        want, _ = plain(x.cpu().double(), [{n: t.cpu().double() for n, t in w.items()} for w in ws])
        close(torch.cat(parts_), want[0], 3.2e-4)
