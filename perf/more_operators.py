"""Linear attention with a decay for each head, and the norms around such a layer: the sizes, types
and options that they are used with.

Three operators. ``op`` "decay": S_t = exp(g_t) S_{t-1} + k_t v_t^T and o_t = scale q_t S_t for each
head, a group of query heads sharing each key head. ``op`` "gated": the norm of a layer's heads (or of
its whole width) with its weight and its gate, before the output projection. ``op`` "residual": the norm
after a block (or none), its scale, the sum with the residual and the norm before the next block.
A case is a dict of plain values:
  kind   "forward"  a prompt or a frozen model: the call without autograd
         "train"    the call under autograd and its gradients, as a training step has it
         "prefill"  packed prompts of a serving batch (ragged lengths, B of them, T tokens in all)
         "decode"   one token per request (B requests, T is 1)
  dtype  the type of q, k and v, or of x, and of the operator's output: "bf16" or "fp32"
  B, T   batch and tokens
decay:
  Hq, H, D  query heads, key and value heads (each serves Hq / H query heads), head dimension
  gate      "token": log-decays (B, T, H); "head": one constant per head, (H,)
  s0        whether the call starts from a state
  view      whether q, k and v are parts of one projection's output
gated:
  H, C       rows of a token (heads) and their width
  gate       the gate's type
  act        "silu" or "sigmoid"
  first      whether the gate comes before the norm
  weight     whether the norm has a weight
  view       whether the gate is a part of a wider projection's output
residual:
  C          channels
  stream     the type of the residual
  post       whether the block's output is normalised (with a weight) before the sum
  scale      what the block's output is multiplied by

Inputs: unit keys and queries and normal values; a head's decay rate is spread over [0.001, 1] by its
logarithm, each token's log-decay is minus that rate times 2 sigmoid(N(0, 1)); states and all other
tensors normal, weights near one.
"""

import math

import numpy as np
import torch

own = False  # False: the plain forms below; True: the framework's entry points


def _decay(name, kind, dtype, B, T, Hq, H, D, gate="token", s0=False, view=False):
    return {"name": name, "op": "decay", "kind": kind, "dtype": dtype, "B": B, "T": T, "Hq": Hq, "H": H, "D": D,
            "gate": gate, "s0": s0, "view": view}


def _gated(name, kind, dtype, B, T, H, C, gate="bf16", act="silu", first=False, weight=True, view=False):
    return {"name": name, "op": "gated", "kind": kind, "dtype": dtype, "B": B, "T": T, "H": H, "C": C, "gate": gate,
            "act": act, "first": first, "weight": weight, "view": view}


def _residual(name, kind, dtype, B, T, C, stream="bf16", post=False, scale=1.0):
    return {"name": name, "op": "residual", "kind": kind, "dtype": dtype, "B": B, "T": T, "C": C, "stream": stream,
            "post": post, "scale": scale}


def listed():
    return [
        # one user decoding: launches and latency only
        _decay("decay decode one request", "decode", "bf16", 1, 1, 16, 16, 128, s0=True),
        # a full batch decoding through the cache's slots, four query heads to a state
        _decay("decay decode full batch", "decode", "bf16", 256, 1, 32, 8, 128, s0=True),
        # prompts of a batch, read from the projection
        _decay("decay prompts bf16", "forward", "bf16", 4, 4096, 16, 16, 128, view=True),
        # one long prompt of a narrow layer, continued from a state: the fewest heads, constant decays
        _decay("decay long prompt bf16", "forward", "bf16", 1, 65521, 8, 4, 128, gate="head", s0=True),
        # ragged prompts packed into one call, into the cache's slots
        _decay("decay packed prompts bf16", "prefill", "bf16", 10, 16384, 16, 16, 128, s0=True),
        # a training step
        _decay("decay train bf16", "train", "bf16", 4, 4096, 16, 16, 128),
        # truncated backpropagation in fp32 over ragged sizes: shared key heads, constant decays, from a state
        _decay("decay train fp32 ragged", "train", "fp32", 3, 1003, 6, 2, 80, gate="head", s0=True),
        # a full batch decoding: the heads' outputs on their way into the output projection
        _gated("gated norm decode full batch", "decode", "bf16", 256, 1, 32, 128),
        # a training step
        _gated("gated norm train bf16", "train", "bf16", 4, 4096, 16, 128, view=True),
        # one user decoding between two blocks
        _residual("residual norm decode one request", "decode", "bf16", 1, 1, 2560, post=True),
        # a training step of a wide model whose blocks are normalised on both sides
        _residual("residual norm train bf16", "train", "bf16", 4, 4096, 4096, post=True),
        # fp32 training over ragged sizes, scaled residuals
        _residual("residual norm train fp32 ragged", "train", "fp32", 3, 1003, 1001, stream="fp32", scale=0.22),
    ]


def draw(rng):
    """One more case of the same ranges: sizes spread over their logarithm, odd ones among them, at
    most as many elements as the listed training steps."""

    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("decay", "decay", "gated", "residual"))
    kind = rng.choice(("forward", "train", "train", "decode") + (("prefill",) if op == "decay" else ()))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    B = log_int(1, 256) if kind == "decode" else log_int(2, 80) if kind == "prefill" else rng.choice((1, 1, 2, 3, 4, 8))

    def tokens(width):  # of one batch row (of all prompts together), at most 2^25 elements in all
        if kind == "decode":
            return 1
        if kind == "prefill":
            return log_int(2 * B, min(1 << 16, (1 << 25) // width))
        return log_int(1, min(1 << 16, (1 << 25) // (B * width)))

    if op == "decay":
        D = rng.choice((32, 64, 64, 80, 96, 128, 128, 192, 256, 33))
        H = rng.choice((1, 2, 3, 4, 8, 16))
        Hq = H * rng.choice((1, 1, 2, 4))
        c = _decay("", kind, dtype, B, tokens(Hq * D * max(1, D // 128)), Hq, H, D, rng.choice(("token", "token", "head")),
                   kind in ("prefill", "decode") or rng.random() < 0.5, kind == "forward" and rng.random() < 0.5)
    elif op == "gated":
        if rng.random() < 0.6:
            H, C = rng.choice((1, 4, 8, 16, 32)), rng.choice((32, 64, 128, 128, 192, 256, 80, 33))
        else:  # the whole width of the layer is one row
            H, C = 1, log_int(256, 8192)
        c = _gated("", kind, dtype, B, tokens(H * C), H, C, "fp32" if dtype == "fp32" else rng.choice(("bf16", "bf16", "fp32")),
                   rng.choice(("silu", "sigmoid")), rng.random() < 0.3, rng.random() < 0.8, rng.random() < 0.4)
    else:
        C = log_int(64, 8192)
        if rng.random() < 0.7:  # most models are multiples of 64 wide, some are odd
            C = C // 64 * 64
        c = _residual("", kind, dtype, B, tokens(C), C, "fp32" if dtype == "fp32" else rng.choice(("bf16", "fp32")),
                      rng.random() < 0.5, rng.choice((1.0, 1.0, 0.22, 0.5)))
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _lengths(case, seed):
    """Offsets of a packed batch: B ragged prompts, T tokens in all."""
    cuts = np.random.default_rng(seed).uniform(0.1, 1.9, case["B"])
    ends = np.floor(np.cumsum(cuts) / cuts.sum() * case["T"]).astype(np.int64)
    ends[-1] = case["T"]
    return np.concatenate([[0], ends])


def _lead(case):
    return {"prefill": (1, case["T"]), "decode": (case["B"],)}.get(case["kind"], (case["B"], case["T"]))


def _decay_inputs(case, seed):
    B, Hq, H, D, dt = case["B"], case["Hq"], case["H"], case["D"], _TYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    lead = _lead(case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def unit(x):
        return x / torch.sqrt((x * x).sum(-1, keepdim=True))

    q, k, v = unit(normal(*lead, Hq, D)).to(dt), unit(normal(*lead, H, D)).to(dt), normal(*lead, H, D).to(dt)
    if case["view"]:
        q, k, v = torch.cat([q, k, v], -2).split([Hq, H, H], -2)
    rate = torch.exp(torch.rand(H, generator=gen, device="cuda") * math.log(1000.0)) * 1e-3
    g = -rate if case["gate"] == "head" else -2.0 * rate * torch.sigmoid(normal(*lead, H))
    st = {"q": q, "k": k, "v": v, "g": g, "s0": None, "cu": None, "slots": None, "go": None, "gs": None}
    if case["s0"]:
        st["s0"] = normal(B, H, D, D)
    if case["kind"] == "prefill":
        st["cu"] = torch.from_numpy(_lengths(case, seed).astype(np.int32)).cuda()
    if case["kind"] in ("prefill", "decode"):
        # a pool half as large again as the batch, which sits on a random part of its slots
        n = B + B // 2 + 1
        st["slots"] = torch.from_numpy(np.sort(np.random.default_rng(seed).permutation(n)[:B]).astype(np.int32)).cuda()
    if case["kind"] == "train":
        st["go"], st["gs"] = normal(*lead, Hq, D).to(dt), normal(B, H, D, D)
    return st


def _gated_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    shape = (*_lead(case), case["H"], case["C"])

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    dt = _TYPES[case["dtype"]]
    z = normal(*shape[:-2], 2 * case["H"] if case["view"] else case["H"], case["C"]).to(_TYPES[case["gate"]])
    return {"x": normal(*shape).to(dt), "z": z[..., z.shape[-2] - case["H"]:, :],
            "w": 1.0 + 0.1 * normal(case["C"]) if case["weight"] else None,
            "gy": normal(*shape).to(dt) if case["kind"] == "train" else None}


def _residual_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    shape = (*_lead(case), case["C"])

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    dt, rt = _TYPES[case["dtype"]], _TYPES[case["stream"]]
    train = case["kind"] == "train"
    return {"x": normal(*shape).to(dt), "r": normal(*shape).to(rt), "w": 1.0 + 0.1 * normal(case["C"]),
            "wp": 1.0 + 0.1 * normal(case["C"]) if case["post"] else None,
            "gy": normal(*shape).to(dt) if train else None, "gh": normal(*shape).to(rt) if train else None}


_INPUTS = {"decay": _decay_inputs, "gated": _gated_inputs, "residual": _residual_inputs}


def prepare(case, seed):
    st = {"case": case, **_INPUTS[case["op"]](case, seed)}
    if st.get("slots") is not None:
        n = case["B"] + case["B"] // 2 + 1
        if own:
            from prometheus_amd import serving
            st["cache"] = serving.DecayStateCache(1, n, case["H"], case["D"])
            st["pool"] = st["cache"].pool[0]
        else:
            st["pool"] = torch.zeros(n, case["H"], case["D"], case["D"], device="cuda")
        st["pool"][st["slots"].long()] = st["s0"]
    if own and case["kind"] == "train":
        for n in ("q", "k", "v", "g", "s0", "x", "z", "w", "r", "wp"):
            if st.get(n) is not None:
                st[n].requires_grad_(True)
    return st


# ---------------------------------------------------------------- the plain forms

_CHUNK = 64


def _chunks(x, n):
    """(N, T, ...) as (N, chunks, 64, ...), zeros behind the last token."""
    pad = torch.zeros((x.shape[0], n * _CHUNK - x.shape[1], *x.shape[2:]), dtype=x.dtype, device=x.device)
    return torch.cat([x, pad], 1).unflatten(1, (n, _CHUNK))


def _between(total):
    """exp of the log-decays between chunks: [.., c, e] is that of the chunks c' with e <= c' < c
    (0 where e > c), from their sums (.., chunks)."""
    ends = torch.cumsum(total, -1)
    starts = torch.cat([torch.zeros_like(ends[..., :1]), ends], -1)
    diff = starts[..., :, None] - starts[..., None, :]
    n = starts.shape[-1]
    keep = torch.ones(n, n, dtype=torch.bool, device=total.device).tril()
    return torch.exp(torch.where(keep, diff, float("-inf"))).float()


def _chunked(q, k, v, g, s0, scale, go=None, gs=None):
    """The operator over (N, T) sequences in chunks of 64 tokens: everything between two tokens of a
    chunk as a (64, 64) matrix, everything else through the states between chunks. With go and gs the
    gradients too. g: (N, T, H) in 64 bits; all else fp32."""
    N, T, Hq, D = q.shape
    H = k.shape[2]
    G, n = Hq // H, -(-T // _CHUNK)
    q, k, v, g = (_chunks(x, n) for x in (q.unflatten(2, (H, G)), k, v, g))
    q = q.permute(0, 3, 1, 4, 2, 5)  # N, H, chunks, G, 64, D
    k, v = (x.permute(0, 3, 1, 2, 4) for x in (k, v))  # N, H, chunks, 64, D
    g = g.permute(0, 3, 1, 2)  # N, H, chunks, 64
    cum = torch.cumsum(g, -1)
    lower = torch.ones(_CHUNK, _CHUNK, dtype=torch.bool, device=q.device).tril()
    pair = torch.exp(torch.where(lower, cum[..., :, None] - cum[..., None, :], float("-inf"))).float()
    into = torch.exp(cum).float()[..., None]  # from the chunk's start to each token
    out_of = torch.exp(cum[..., -1:] - cum).float()[..., None]  # from each token to the chunk's end
    total = cum[..., -1]
    across = _between(total)  # N, H, chunks + 1, chunks + 1
    s0 = torch.zeros(N, H, D, D, device=q.device) if s0 is None else s0
    own_part = torch.matmul(k.transpose(-1, -2), v * out_of).flatten(-2)  # each chunk's own share of the state
    states = torch.matmul(across[..., 1:], own_part) + across[..., :1] * s0.flatten(-2)[:, :, None]
    states = states.unflatten(-1, (D, D))  # before each chunk, and the last one
    before = states[:, :, :-1]
    # (a product batched over the group, its rows under one another)
    scores = torch.matmul(q.flatten(3, 4), k.transpose(-1, -2)).unflatten(3, (G, _CHUNK))
    masked = scores * pair[:, :, :, None]
    o = torch.matmul(masked.flatten(3, 4), v).unflatten(3, (G, _CHUNK))
    o = scale * (o + into[:, :, :, None] * torch.matmul(q.flatten(3, 4), before).unflatten(3, (G, _CHUNK)))

    def rows(x):  # N, H, chunks, (G,) 64, D back to N, T, heads, D
        x = x.permute(0, 2, 4, 1, 3, 5) if x.dim() == 6 else x.permute(0, 2, 3, 1, 4)
        return x.reshape(N, n * _CHUNK, -1, D)[:, :T]

    if go is None:
        return rows(o), states[:, :, -1]
    go = _chunks(go.unflatten(2, (H, G)), n).permute(0, 3, 1, 4, 2, 5) * scale
    # the gradient of the state after each chunk: the sums run from the last chunk to the first
    back = torch.matmul((q * into[:, :, :, None]).flatten(3, 4).transpose(-1, -2), go.flatten(3, 4)).flatten(-2)
    across_t = across.transpose(-1, -2)
    after = torch.matmul(across_t[..., :-1], back) + across_t[..., -1:] * gs.flatten(-2)[:, :, None]
    after = after.unflatten(-1, (D, D))
    ds0, after = after[:, :, 0], after[:, :, 1:]
    gscores = torch.matmul(go.flatten(3, 4), v.transpose(-1, -2)).unflatten(3, (G, _CHUNK))
    gmasked = gscores * pair[:, :, :, None]
    dq_far = into[:, :, :, None] * torch.matmul(go.flatten(3, 4), before.transpose(-1, -2)).unflatten(3, (G, _CHUNK))
    dk_far = out_of * torch.matmul(v, after.transpose(-1, -2))
    dq = torch.matmul(gmasked.flatten(3, 4), k).unflatten(3, (G, _CHUNK)) + dq_far
    dk = torch.matmul(gmasked.flatten(3, 4).transpose(-1, -2), q.flatten(3, 4)) + dk_far
    dv = torch.matmul(masked.flatten(3, 4).transpose(-1, -2), go.flatten(3, 4)) + out_of * torch.matmul(k, after)
    # dL/dg_t: everything that passes from before token t to it or later ones
    passing = (scores * gmasked).sum(3)  # [i, j] of a chunk
    left = torch.cumsum(passing, -1) - passing  # [i, t]: the sum over j < t
    near = torch.where(lower, left, 0.0).sum(-2)
    r, c = (q * dq_far).sum((3, 5)), (k * dk_far).sum(-1)
    r_on = torch.flip(torch.cumsum(torch.flip(r, (-1,)), -1), (-1,))
    c_before = torch.cumsum(c, -1) - c
    whole = torch.exp(total).float() * (before * after).sum((-1, -2))
    dg = (near + r_on + c_before + whole[..., None]).permute(0, 2, 3, 1).reshape(N, n * _CHUNK, H)[:, :T]
    return rows(o), states[:, :, -1], rows(dq), rows(dk), rows(dv), dg, ds0


def _plain_decay(st):
    case, dt = st["case"], st["q"].dtype
    B, T, Hq, H, D = (case[n] for n in ("B", "T", "Hq", "H", "D"))
    scale = 1.0
    q, k, v = (st[n].float() for n in ("q", "k", "v"))
    g = st["g"].double().expand(*st["q"].shape[:-2], H)
    if case["kind"] == "decode":
        slots = st["slots"].long()
        s = torch.exp(g).float()[..., None, None] * st["pool"][slots] + k[..., :, None] * v[..., None, :]
        st["pool"][slots] = s
        o = torch.matmul(q.unflatten(1, (H, Hq // H)), s).flatten(1, 2)
        return {"o": (scale * o).to(dt), "pool": st["pool"]}
    if case["kind"] == "prefill":
        # each prompt a row of its own, as long as the longest
        slots, cu = st["slots"].long(), st["cu"].long()
        first, length = cu[:-1, None], (cu[1:] - cu[:-1])[:, None]
        at = torch.arange(int(length.max()), device="cuda")[None]
        there = at < length
        index = torch.where(there, first + at, 0)
        keep = there[..., None, None]
        o, s = _chunked(q[0][index] * keep, k[0][index] * keep, v[0][index] * keep, g[0][index] * there[..., None],
                        st["pool"][slots], scale)
        st["pool"][slots] = s
        return {"o": o[there][None].to(dt), "pool": st["pool"]}
    if case["kind"] == "forward":
        o, s = _chunked(q, k, v, g, st["s0"], scale)
        return {"o": o.to(dt), "state": s.clone()}
    o, s, dq, dk, dv, dg, ds0 = _chunked(q, k, v, g, st["s0"], scale, st["go"].float(), st["gs"])
    out = {"o": o.to(dt), "state": s.clone(), "dq": dq.to(dt), "dk": dk.to(dt), "dv": dv.to(dt),
           "dg": dg.double().sum((0, 1)).float() if case["gate"] == "head" else dg.clone()}
    if st["s0"] is not None:
        out["ds0"] = ds0.clone()
    return out


_EPS = 1e-6


def _plain_gated(st):
    case, x, z, w = st["case"], st["x"].float(), st["z"].float(), st["w"]
    sig = 1.0 / (1.0 + torch.exp(-z))
    a = z * sig if case["act"] == "silu" else sig
    u = x * a if case["first"] else x
    r = 1.0 / torch.sqrt((u * u).mean(-1, keepdim=True) + _EPS)
    n = u * r
    weighted = n if w is None else n * w
    y = weighted if case["first"] else weighted * a
    out = {"y": y.to(st["x"].dtype)}
    if st["gy"] is not None:
        gy = st["gy"].float()
        slope = sig * (1.0 - sig)
        slope = sig + z * slope if case["act"] == "silu" else slope
        gn = gy if case["first"] else gy * a
        if w is not None:
            out["dw"] = (gn * n).sum(tuple(range(x.dim() - 1)))
            gn = gn * w
        gu = r * (gn - n * (gn * n).mean(-1, keepdim=True))
        out["dx"] = (gu * a if case["first"] else gu).to(st["x"].dtype)
        out["dz"] = ((gu * x if case["first"] else gy * weighted) * slope).to(st["z"].dtype)
    return out


def _plain_residual(st):
    case, x, res, w, wp = st["case"], st["x"].float(), st["r"].float(), st["w"], st["wp"]
    if wp is None:
        b = x
    else:
        rp = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS)
        np_ = x * rp
        b = np_ * wp
    h = res + case["scale"] * b
    r = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + _EPS)
    n = h * r
    out = {"y": (n * w).to(st["x"].dtype), "h": h.to(st["r"].dtype)}
    if st["gy"] is not None:
        lead = tuple(range(x.dim() - 1))
        gn = st["gy"].float()
        out["dw"] = (gn * n).sum(lead)
        gn = gn * w
        dh = st["gh"].float() + r * (gn - n * (gn * n).mean(-1, keepdim=True))
        gb = case["scale"] * dh
        if wp is not None:
            out["dwp"] = (gb * np_).sum(lead)
            gb = gb * wp
            gb = rp * (gb - np_ * (gb * np_).mean(-1, keepdim=True))
        out["dx"], out["dr"] = gb.to(st["x"].dtype), dh.to(st["r"].dtype)
    return out


# ---------------------------------------------------------------- one pass


def _gradients(st, out, outputs, names, grads):
    names = [n for n in names if st[n] is not None]
    got = torch.autograd.grad(outputs, [st[n] for n in names], grads)
    out.update({"d" + n: g for n, g in zip(names, got)})
    return out


def _own_decay(st):
    from prometheus_amd import kernels
    case, dt = st["case"], st["q"].dtype
    qkv = st["q"], st["k"], st["v"]
    if case["kind"] == "decode":
        return {"o": st["cache"].decode(0, st["slots"], *qkv, st["g"], out_dtype=dt), "pool": st["pool"]}
    if case["kind"] == "prefill":
        o = st["cache"].prefill(0, st["slots"], *qkv, st["g"], st["cu"], out_dtype=dt)
        return {"o": o, "pool": st["pool"]}
    o, s = kernels.decay_attention(*qkv, st["g"], st["s0"], out_dtype=dt)
    out = {"o": o.detach(), "state": s.detach()}
    if case["kind"] == "train":
        _gradients(st, out, (o, s), ("q", "k", "v", "g", "s0"), (st["go"], st["gs"]))
    return out


def _own_gated(st):
    from prometheus_amd import kernels
    case = st["case"]
    y = kernels.gated_norm(st["x"], st["z"], st["w"], activation=case["act"], gate_first=case["first"],
                           out_dtype=st["x"].dtype)
    out = {"y": y.detach()}
    return _gradients(st, out, (y,), ("x", "z", "w"), (st["gy"],)) if case["kind"] == "train" else out


def _own_residual(st):
    from prometheus_amd import kernels
    case = st["case"]
    y, h = kernels.residual_norm(st["x"], st["r"], st["w"], post_weight=st["wp"], scale=case["scale"])
    out = {"y": y.detach(), "h": h.detach()}
    if case["kind"] == "train":
        _gradients(st, out, (y, h), ("x", "r", "w", "wp"), (st["gy"], st["gh"]))
    return out


def run(st):
    op = st["case"]["op"]
    if own:
        return {"decay": _own_decay, "gated": _own_gated, "residual": _own_residual}[op](st)
    return {"decay": _plain_decay, "gated": _plain_gated, "residual": _plain_residual}[op](st)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    """The forward's inputs read once and its outputs written once; a training pass adds the same of
    the backward, a call of its own that comes after the rest of the model has run."""
    e = 2 if case["dtype"] == "bf16" else 4
    B, train = case["B"], case["kind"] == "train"
    tokens = case["T"] if case["kind"] == "prefill" else B * case["T"]
    if case["op"] == "decay":
        Hq, H, D = case["Hq"], case["H"], case["D"]
        gates = 4 * H * (1 if case["gate"] == "head" else tokens)
        state = 4 * B * H * D * D
        nbytes = tokens * D * e * (2 * Hq + 2 * H) + gates + state * (2 if case["s0"] else 1)
        flops = 2.0 * tokens * D * D * (H + Hq)  # the state's update for each key head, its product for each query head
        if train:  # q, k, v, go and gs in; gq, gk, gv, gg (and the first state's) out
            nbytes += tokens * D * e * (3 * Hq + 4 * H) + 2 * gates + state * (3 if case["s0"] else 1)
            flops += 2.0 * tokens * D * D * (2 * Hq + 3 * H)
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "gated":
        n, eg = tokens * case["H"] * case["C"], 2 if case["gate"] == "bf16" else 4
        w = 4 * case["C"] if case["weight"] else 0
        nbytes, flops = n * (2 * e + eg) + w, 8.0 * n
        if train:  # x, the gate and gy in; gx and the gate's gradient out
            nbytes += n * (3 * e + 2 * eg) + 2 * w
            flops += 20.0 * n
        return {"bytes": nbytes, "flops": flops}
    n, er = tokens * case["C"], 2 if case["stream"] == "bf16" else 4
    w = 4 * case["C"] * (2 if case["post"] else 1)
    nbytes, flops = n * (2 * e + 2 * er) + w, 10.0 * n
    if train:  # x, the residual, gy and gh in; gx and the residual's gradient out
        nbytes += n * (3 * e + 3 * er) + 2 * w
        flops += 24.0 * n
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------- the same in 64 bits


def _walk(q, k, v, g, s, go=None):
    """Token by token over (N, T, H, ...) in 64 bits from the states s (N, H, D, D): the outputs, and
    with go the products S_t go_t (q's gradients)."""
    o = torch.empty_like(q)
    dq = None if go is None else torch.empty_like(q)
    G = q.shape[2] // k.shape[2]
    s = s.clone()
    a = torch.exp(g)
    for t in range(q.shape[1]):
        s *= a[:, t, :, None, None]
        s += k[:, t, :, :, None] * v[:, t, :, None, :]
        o[:, t] = (q[:, t].unflatten(1, (-1, G))[..., None, :] @ s[:, :, None]).flatten(1, 3).view_as(o[:, t])
        if go is not None:
            dq[:, t] = (s[:, :, None] @ go[:, t].unflatten(1, (-1, G))[..., None]).flatten(1, 2)[..., 0]
    return o, s, dq


def _exact_decay(case, seed):
    st = _decay_inputs(case, seed)
    f64 = torch.float64
    B, H, D = case["B"], case["H"], case["D"]
    q, k, v = (st[n].double() for n in ("q", "k", "v"))
    g = st["g"].double().expand(*q.shape[:-2], H)
    if case["kind"] in ("decode", "prefill"):
        slots = st["slots"].long()
        pool = torch.zeros(B + B // 2 + 1, H, D, D, device="cuda", dtype=f64)
        pool[slots] = st["s0"].double()
        if case["kind"] == "decode":
            o, s, _ = _walk(q[:, None], k[:, None], v[:, None], g[:, None], pool[slots])
            pool[slots] = s
            return {"o": o[:, 0], "pool": pool}
        o, cu = torch.empty_like(q), st["cu"].tolist()
        for i, (a, z) in enumerate(zip(cu[:-1], cu[1:])):
            o[:, a:z], pool[slots[i]], _ = _walk(q[:, a:z], k[:, a:z], v[:, a:z], g[:, a:z], pool[slots[i]][None])
        return {"o": o, "pool": pool}
    s0 = torch.zeros(B, H, D, D, device="cuda", dtype=f64) if st["s0"] is None else st["s0"].double()
    if case["kind"] == "forward":
        o, s, _ = _walk(q, k, v, g, s0)
        return {"o": o, "state": s}
    go, d = st["go"].double(), st["gs"].double().clone()
    o, s, dq = _walk(q, k, v, g, s0, go)
    G = case["Hq"] // H
    last = (s * d).sum((-1, -2))
    dk, dv = torch.empty_like(k), torch.empty_like(v)
    for t in range(case["T"] - 1, -1, -1):
        d += q[:, t].unflatten(1, (H, G)).transpose(-1, -2) @ go[:, t].unflatten(1, (H, G))
        dk[:, t] = (d @ v[:, t, :, :, None])[..., 0]
        dv[:, t] = (k[:, t, :, None, :] @ d)[..., 0, :]
        d *= torch.exp(g[:, t])[..., None, None]
    # d log of what leaves token t and what enters it: the sums over all later tokens telescope
    flow = (q * dq).sum(-1).unflatten(2, (H, G)).sum(-1) - (k * dk).sum(-1)
    dg = flow.flip(1).cumsum(1).flip(1) + last[:, None]
    out = {"o": o, "state": s, "dq": dq, "dk": dk, "dv": dv, "dg": dg.sum((0, 1)) if case["gate"] == "head" else dg}
    if st["s0"] is not None:
        out["ds0"] = d
    return out


def _leaf(x, train):
    return None if x is None else x.double().requires_grad_(train)


def _exact_norm(names, case, st, operator, outputs, grads):
    """The operator's outputs in 64 bits, and the gradients that autograd makes of its formula."""
    train = case["kind"] == "train"
    x = {n: _leaf(st[n], train) for n in names}
    ys = operator(**x)
    out = {n: y.detach() for n, y in zip(outputs, ys)}
    if train:
        there = [n for n in names if x[n] is not None]
        got = torch.autograd.grad(ys, [x[n] for n in there], [st[n].double() for n in grads])
        out.update({"d" + n: v for n, v in zip(there, got)})
    return out


def _rms(u):
    return u * torch.rsqrt(u.square().mean(-1, keepdim=True) + _EPS)


def _exact_gated(case, seed):
    def operator(x, z, w):
        a = torch.nn.functional.silu(z) if case["act"] == "silu" else torch.sigmoid(z)
        w = 1.0 if w is None else w
        return (_rms(x * a) * w if case["first"] else _rms(x) * w * a,)

    return _exact_norm(("x", "z", "w"), case, _gated_inputs(case, seed), operator, ("y",), ("gy",))


def _exact_residual(case, seed):
    def operator(x, r, w, wp):
        h = r + case["scale"] * (x if wp is None else _rms(x) * wp)
        return _rms(h) * w, h

    return _exact_norm(("x", "r", "w", "wp"), case, _residual_inputs(case, seed), operator, ("y", "h"), ("gy", "gh"))


def exact(case, seed):
    return {"decay": _exact_decay, "gated": _exact_gated, "residual": _exact_residual}[case["op"]](case, seed)
