"""64-bit CPU forms of the operators beside the delta rule, and bounds on their fp32 errors.

The recurrence ``h_t = exp(g_t) h_{t-1} + x_t`` and the heads' norms with the position rotation,
each with its gradients from the formulas, token by token and pair by pair in NumPy. The ``*_bound``
functions say how far an fp32 computation may be off, from the roundings on each term's way.
"""

from __future__ import annotations

import numpy as np

U32 = 2.0**-24  # half a step of fp32


def recurrence(x, g, s0=None):
    """(B, T, C) arrays: ``(h, state)``."""
    x, a = np.asarray(x, np.float64), np.exp(np.asarray(g, np.float64))
    s = np.zeros((x.shape[0], x.shape[2])) if s0 is None else np.asarray(s0, np.float64)
    h = np.empty_like(x)
    for t in range(x.shape[1]):
        s = a[:, t] * s + x[:, t]
        h[:, t] = s
    return h, s


def recurrence_bwd(x, g, s0, gh, gs):
    """``(gx, gg, gs0)`` of ``sum(gh h) + sum(gs state)``."""
    h, _ = recurrence(x, g, s0)
    a = np.exp(np.asarray(g, np.float64))
    gx, gg = np.zeros_like(h), np.zeros_like(h)
    start = np.zeros_like(h[:, 0]) if s0 is None else np.asarray(s0, np.float64)
    carry = np.zeros_like(start) if gs is None else np.asarray(gs, np.float64)
    for t in range(h.shape[1] - 1, -1, -1):
        d = carry if gh is None else np.asarray(gh, np.float64)[:, t] + carry
        carry = a[:, t] * d
        gx[:, t], gg[:, t] = d, carry * (h[:, t - 1] if t else start)
    return gx, gg, carry


def recurrence_bound(x, g, s0=None):
    """How far fp32 may be off h, per element. Each term x_s exp(g_{s+1} + .. + g_t) meets, a token,
    one gate and one multiply-add: the gate's relative error is at most 4 + 4 |g| half steps (a
    rounded product of g before the exponential, the exponential itself within a step of the
    hardware's), the multiply-add's one; joining spans adds at most 32 products and sums in all."""
    g = np.asarray(g, np.float64)
    a = np.exp(g)
    big, _ = recurrence(np.abs(np.asarray(x, np.float64)), g, None if s0 is None else np.abs(s0))
    before = np.concatenate([np.zeros_like(big[:, :1]) if s0 is None else np.abs(np.asarray(s0, np.float64))[:, None],
                             big[:, :-1]], 1)
    each = U32 * ((5.0 + 4.0 * np.abs(g)) * a * before + big)
    off, _ = recurrence(each, g)
    return off + 32 * U32 * big


def recurrence_bwd_bound(x, g, s0, gh, gs):
    """How far fp32 may be off ``(gx, gg, gs0)``: gx is the same recurrence from the last token to
    the first; gg multiplies it by the recomputed state before."""
    x, g = np.asarray(x, np.float64), np.asarray(g, np.float64)
    B, T, C = x.shape
    a = np.exp(g)
    ghd = np.zeros_like(x) if gh is None else np.asarray(gh, np.float64)
    gsd = np.zeros((B, C)) if gs is None else np.asarray(gs, np.float64)
    # d_t = gh_t + a_{t+1} d_{t+1} with gs as the carry into the last token
    nxt = np.concatenate([g[:, 1:], np.zeros((B, 1, C))], 1)[:, ::-1]
    big, _ = recurrence(np.abs(ghd)[:, ::-1], nxt, np.abs(gsd))
    off_d = recurrence_bound(ghd[:, ::-1], nxt, gsd)[:, ::-1]
    big = big[:, ::-1]
    h, _ = recurrence(np.abs(x), g, None if s0 is None else np.abs(s0))
    off_h = recurrence_bound(x, g, s0)
    start = np.zeros((B, 1, C)) if s0 is None else np.abs(np.asarray(s0, np.float64))[:, None]
    before = np.concatenate([start, h[:, :-1]], 1)
    off_before = np.concatenate([np.zeros((B, 1, C)), off_h[:, :-1]], 1)
    gate = U32 * (5.0 + 4.0 * np.abs(g))
    off_g = a * (off_d * before + big * off_before + big * before * (gate + 3 * U32))
    off_s = a[:, 0] * (off_d[:, 0] + big[:, 0] * gate[:, 0]) if T else np.zeros((B, C))
    return off_d, off_g, off_s


def _pairs(R, interleaved):
    i = np.arange(R // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)


def _turn(y, cos, sin, interleaved):
    first, second = _pairs(2 * cos.shape[-1], interleaved)
    z = y.copy()
    z[..., first] = y[..., first] * cos - y[..., second] * sin
    z[..., second] = y[..., second] * cos + y[..., first] * sin
    return z


def _angles(table, positions):
    rows = np.asarray(table, np.float64)[positions]
    half = rows.shape[-1] // 2
    return rows[..., None, :half], rows[..., None, half:]


def _unit(x, norm, eps):
    """``(u, r, clipped)``: u = r x."""
    ss = np.sum(x * x, -1, keepdims=True)
    if norm == "l2":
        n = np.sqrt(ss)
        r, clipped = 1.0 / np.maximum(n, eps), n <= eps
    else:
        r, clipped = 1.0 / np.sqrt(ss / x.shape[-1] + eps), np.zeros(ss.shape, bool)
    return x * r, r, clipped


def head_norm(x, table=None, positions=None, norm="l2", weight=None, eps=1e-6, interleaved=False):
    """One of q and k, (..., H, D); positions (...,)."""
    u, _, _ = _unit(np.asarray(x, np.float64), norm, eps)
    y = u if weight is None else u * np.asarray(weight, np.float64)
    return y if table is None else _turn(y, *_angles(table, positions), interleaved)


def head_norm_bwd(x, gz, table=None, positions=None, norm="l2", weight=None, eps=1e-6, interleaved=False):
    """``(gx, gweight)`` of ``sum(gz head_norm(x))``."""
    x, gy = np.asarray(x, np.float64), np.asarray(gz, np.float64)
    u, r, clipped = _unit(x, norm, eps)
    if table is not None:
        cos, sin = _angles(table, positions)
        gy = _turn(gy, cos, -sin, interleaved)
    gw = np.sum((gy * u).reshape(-1, x.shape[-1]), 0)
    gu = gy if weight is None else gy * np.asarray(weight, np.float64)
    dot = np.sum(gu * u, -1, keepdims=True) / (x.shape[-1] if norm == "rms" else 1)
    return r * (gu - np.where(clipped, 0.0, u * dot)), gw


def _turn_sizes(y, table, positions, interleaved):
    """|y1 cos| + |y2 sin| and |y2 cos| + |y1 sin| for y >= 0."""
    cos, sin = (np.abs(t) for t in _angles(table, positions))
    first, second = _pairs(2 * cos.shape[-1], interleaved)
    z = y.copy()
    z[..., first] = y[..., first] * cos + y[..., second] * sin
    z[..., second] = y[..., second] * cos + y[..., first] * sin
    return z


def head_norm_bound(x, table=None, positions=None, norm="l2", weight=None, eps=1e-6, interleaved=False):
    """How far fp32 may be off head_norm: the sum of D <= 256 squares in a tree over lanes and
    registers (at most 16 roundings, halved by the root), root, division, products: 24 half steps
    of each of the two terms of an element."""
    u, _, _ = _unit(np.abs(np.asarray(x, np.float64)), norm, eps)
    y = u if weight is None else u * np.abs(np.asarray(weight, np.float64))
    if table is not None:
        y = _turn_sizes(y, table, positions, interleaved)
    return 24 * U32 * y + 1e-30


def head_norm_bwd_bound(x, gz, table=None, positions=None, norm="l2", weight=None, eps=1e-6, interleaved=False):
    """How far fp32 may be off head_norm_bwd: 40 half steps of each term's size for gx (as above,
    the turn back, the dot product over D and two products); for the weights' gradient the terms'
    own error and one rounding per row summed."""
    x, gz = np.abs(np.asarray(x, np.float64)), np.abs(np.asarray(gz, np.float64))
    u, r, _ = _unit(x, norm, eps)
    gy = gz if table is None else _turn_sizes(gz, table, positions, interleaved)
    terms = (gy * u).reshape(-1, x.shape[-1])
    gu = gy if weight is None else gy * np.abs(np.asarray(weight, np.float64))
    dot = np.sum(gu * u, -1, keepdims=True) / (x.shape[-1] if norm == "rms" else 1)
    return 40 * U32 * r * (gu + u * dot) + 1e-30, (40 + len(terms)) * U32 * terms.sum(0) + 1e-30
