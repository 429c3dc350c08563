"""Plain 64-bit forms of linear attention with a decay for each head, token by token, and of the norms
around such a layer: what their tests compare with. CPU tensors in, CPU float64 tensors out."""

from __future__ import annotations

import torch

F64 = torch.float64


def _per_token(g, q, H):
    return g.to(F64).expand(*q.shape[:2], H)


def decay(q, k, v, g, s0=None, scale=1.0):
    """``(o, state)`` of q (B, T, Hq, D), k, v (B, T, H, D), g (B, T, H) or (H,)."""
    q, k, v = (x.to(F64) for x in (q, k, v))
    (B, T, Hq, D), H = q.shape, k.shape[2]
    g = _per_token(g, q, H)
    s = torch.zeros(B, H, D, D, dtype=F64) if s0 is None else s0.to(F64).clone()
    o = torch.empty(q.shape, dtype=F64)
    for t in range(T):
        s = torch.exp(g[:, t])[..., None, None] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        o[:, t] = scale * torch.einsum("bhgd,bhde->bhge", q[:, t].unflatten(1, (H, Hq // H)), s).flatten(1, 2)
    return o, s


def decay_bwd(q, k, v, g, s0, go, gs, scale=1.0):
    """``(gq, gk, gv, gg, gs0)``; gg like g. Every gradient of a log-decay is the product of the state
    before the token and the gradient of the state after it: no sums telescope."""
    q, k, v, go = (x.to(F64) for x in (q, k, v, go))
    (B, T, Hq, D), H = q.shape, k.shape[2]
    shape, g = g.shape, _per_token(g, q, H)
    a = torch.exp(g)[..., None, None]
    s = torch.zeros(B, H, D, D, dtype=F64) if s0 is None else s0.to(F64).clone()
    qg, gog = q.unflatten(2, (H, Hq // H)), go.unflatten(2, (H, Hq // H))
    decayed, gq = [], torch.empty(qg.shape, dtype=F64)
    for t in range(T):
        decayed.append(a[:, t] * s)
        s = decayed[-1] + k[:, t, :, :, None] * v[:, t, :, None, :]
        gq[:, t] = scale * torch.einsum("bhde,bhge->bhgd", s, gog[:, t])
    d = torch.zeros_like(s) if gs is None else gs.to(F64).clone()
    gk, gv, gg = torch.empty_like(k), torch.empty_like(v), torch.empty(B, T, H, dtype=F64)
    for t in reversed(range(T)):
        d = d + scale * torch.einsum("bhgd,bhge->bhde", qg[:, t], gog[:, t])
        gk[:, t] = torch.einsum("bhde,bhe->bhd", d, v[:, t])
        gv[:, t] = torch.einsum("bhde,bhd->bhe", d, k[:, t])
        gg[:, t] = (d * decayed[t]).sum((-1, -2))
        d = a[:, t] * d
    return gq.flatten(2, 3), gk, gv, gg.sum((0, 1)) if len(shape) == 1 else gg, d


def gated(x, z, w=None, activation="silu", gate_first=False, eps=1e-6):
    x, z = x.to(F64), z.to(F64)
    a = torch.sigmoid(z) * (z if activation == "silu" else 1.0)
    u = x * a if gate_first else x
    y = u / torch.sqrt((u * u).mean(-1, keepdim=True) + eps) * (1.0 if w is None else w.to(F64))
    return y if gate_first else y * a


def residual(x, r, w=None, wp=None, scale=1.0, eps=1e-6):
    x, r = x.to(F64), r.to(F64)
    b = x if wp is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * wp.to(F64)
    h = r + scale * b
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * (1.0 if w is None else w.to(F64)), h


def _rms_bwd_size(p, u, eps):
    """The absolute terms of r (p - n mean(p n)), n = r u, and n, for |p|."""
    r = 1.0 / torch.sqrt((u * u).mean(-1, keepdim=True) + eps)
    n = (r * u).abs()
    return r * (p + n * (p * n).mean(-1, keepdim=True)), n


def gated_bwd_size(x, z, w, gy, activation="silu", gate_first=False, eps=1e-6):
    """The terms of gx, gz and gw with absolute values: what their rounding errors are relative to."""
    x, z, gy = x.to(F64), z.to(F64), gy.to(F64).abs()
    w = torch.ones(x.shape[-1], dtype=F64) if w is None else w.to(F64).abs()
    s = torch.sigmoid(z)
    a = (s * (z if activation == "silu" else 1.0)).abs()
    slope = s + (z * s * (1 - s)).abs() if activation == "silu" else s * (1 - s)
    g = gy if gate_first else gy * a
    gu, n = _rms_bwd_size(g * w, x * a if gate_first else x, eps)
    gz = (gu * x.abs() if gate_first else gy * n * w) * slope
    return gu * a if gate_first else gu, gz, (g * n).flatten(0, -2).sum(0)


def residual_bwd_size(x, r, w, wp, gy, gh, scale=1.0, eps=1e-6):
    """The same of gx, gr, gw and gwp."""
    x, gy, gh = x.to(F64), gy.to(F64).abs(), gh.to(F64).abs()
    w = 1.0 if w is None else w.to(F64).abs()
    _, h = residual(x, r, None, wp, scale, eps)
    dh, n = _rms_bwd_size(gy * w, h, eps)
    dh = dh + gh
    gw = (gy * n).flatten(0, -2).sum(0)
    if wp is None:
        return abs(scale) * dh, dh, gw, None
    gx, m = _rms_bwd_size(abs(scale) * dh * wp.to(F64).abs(), x, eps)
    return gx, dh, gw, (abs(scale) * dh * m).flatten(0, -2).sum(0)


def gradients(f, inputs, grads):
    """The gradients of f's outputs by autograd in 64 bits: None where an input is None."""
    leaves = [None if x is None else x.detach().to(F64).requires_grad_(True) for x in inputs]
    outs = f(*leaves)
    outs = outs if isinstance(outs, tuple) else (outs,)
    loss = sum((o * g.to(F64)).sum() for o, g in zip(outs, grads) if g is not None)
    there = [x for x in leaves if x is not None]
    got = iter(torch.autograd.grad(loss, there, allow_unused=True))
    return [None if x is None else next(got) for x in leaves]


def planes(x, n):
    """x as the sum of its first n bf16 parts: the value rounded, what that leaves rounded, and so on."""
    rest, out = x.to(F64), torch.zeros_like(x, dtype=F64)
    for _ in range(n):
        part = rest.float().bfloat16().to(F64)
        out, rest = out + part, rest - part
    return out


def chunked(q, k, v, g, s0=None, scale=1.0, chunk=64, inputs=None, factors=None, decayed=None):
    """``decay`` in chunks, in 64 bits but for the factors of its products, which are sums of so many bf16
    parts (None: as they are): of the inputs, of the state and of A = e^{G_i - G_j} q_i . k_j in what
    comes out, and of the decayed V that enters the state."""
    def cut(x, n):
        return x if n is None else planes(x, n)

    (B, T, Hq, D), H = q.shape, k.shape[2]
    q, k, v = (cut(x.to(F64), inputs) for x in (q, k, v))
    g = _per_token(g, q, H)
    s = torch.zeros(B, H, D, D, dtype=F64) if s0 is None else s0.to(F64).clone()
    o = torch.empty(q.shape, dtype=F64)
    for a in range(0, T, chunk):
        z = min(a + chunk, T)
        G = torch.cumsum(g[:, a:z], 1).transpose(1, 2)  # B, H, C
        qc, kc, vc = (x[:, a:z].transpose(1, 2) for x in (q, k, v))
        qc = qc.unflatten(1, (H, Hq // H))  # B, H, group, C, D
        lower = torch.ones(z - a, z - a, dtype=torch.bool).tril()
        pair = torch.exp(torch.where(lower, G[..., :, None] - G[..., None, :], float("-inf")))
        A = cut(scale * (qc @ kc[:, :, None].transpose(-1, -2)) * pair[:, :, None], factors)
        into = scale * torch.exp(G)[:, :, None, :, None] * (qc @ cut(s, factors)[:, :, None])
        o[:, a:z] = (into + A @ vc[:, :, None]).flatten(1, 2).transpose(1, 2)
        s = torch.exp(G[..., -1])[..., None, None] * s + kc.transpose(-1, -2) @ cut(
            vc * torch.exp(G[..., -1:] - G)[..., None], decayed)
    return o, s


def _squares(*xs):
    return [None if x is None else x.to(F64) ** 2 for x in xs]


def spread(q, k, v, g, s0=None, scale=1.0):
    """The root of the sum of squares of the terms of o and of the state: what independent errors of the
    terms, relative to each, come to."""
    return [x.sqrt() for x in decay(*_squares(q, k, v), 2 * g.to(F64), *_squares(s0), scale**2)]


def spread_bwd(q, k, v, g, s0, go, gs, scale=1.0):
    """The same of the gradients (per token, also where g is one constant a head)."""
    g = _per_token(g, q, k.shape[2])
    return [x.sqrt() for x in decay_bwd(*_squares(q, k, v), 2 * g, *_squares(s0, go, gs), scale**2)]


def rms(x):
    return x.to(F64).square().mean().sqrt().item()
