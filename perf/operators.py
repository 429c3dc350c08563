"""The operators beside the delta rule, over the sizes, types and options that they are used with.

Two operators: the elementwise gated linear recurrence (``op`` "recurrence") and the norms of
queries and keys for each head with the position rotation in the same pass (``op`` "heads").
A case is a dict of plain values:
  kind   "forward"  a prompt or a frozen model: the call without autograd
         "train"    the call under autograd and its gradients, as a training step has it
         "prefill"  packed prompts of a serving batch (ragged lengths, B of them, T tokens in all)
         "decode"   one token per request (B requests, T is 1)
  dtype  the type of x, or of q and k: "bf16" or "fp32"; outputs and their gradients have it too
  B, T   batch and tokens
recurrence:
  C      channels
  gate   the type of the log-gates
  s0     whether the call starts from a state
  view   whether x and g are the halves of one projection's output
heads:
  Hq, Hk, D   query heads, key heads, head dimension
  R           rotated dimensions of a head (0: no rotation)
  norm        "l2" or "rms"
  weight      whether each norm has a weight per dimension
  interleaved pairs (2i, 2i + 1) instead of (i, i + R / 2)
  view        whether q and k are parts of one projection's output

Inputs: log-gates -c_j 2 sigmoid(N(0, 1)) with a rate c_j per channel, spread over [0.001, 1] by
its logarithm; x normal, scaled by sqrt(1 - a^2) so that the state stays of order one; q and k
normal, weights near one, positions as prompts and decoding requests have them.
"""

import math

import numpy as np
import torch

own = False  # False: the plain forms below; True: the framework's entry points


def _rec(name, kind, dtype, B, T, C, gate="bf16", s0=False, view=False):
    return {"name": name, "op": "recurrence", "kind": kind, "dtype": dtype, "B": B, "T": T, "C": C,
            "gate": gate, "s0": s0, "view": view}


def _heads(name, kind, dtype, B, T, Hq, Hk, D, R, norm="l2", weight=False, interleaved=False, view=False):
    return {"name": name, "op": "heads", "kind": kind, "dtype": dtype, "B": B, "T": T, "Hq": Hq, "Hk": Hk,
            "D": D, "R": R, "norm": norm, "weight": weight, "interleaved": interleaved, "view": view}


def listed():
    return [
        # one user decoding: launches and latency only
        _rec("recurrence decode one request", "decode", "bf16", 1, 1, 2560, s0=True),
        # a full batch decoding through the cache's slots, gates kept in fp32
        _rec("recurrence decode full batch", "decode", "bf16", 256, 1, 4096, gate="fp32", s0=True),
        # a short fp32 call (tests, references, small models)
        _rec("recurrence short fp32", "forward", "fp32", 1, 77, 512, gate="fp32"),
        # a training step of a wide layer
        _rec("recurrence train bf16", "train", "bf16", 4, 4096, 4096),
        # truncated backpropagation in fp32 over ragged sizes, from a state
        _rec("recurrence train fp32 ragged", "train", "fp32", 3, 1003, 1001, gate="fp32", s0=True),
        # one long prompt of a narrow layer, continued from a state: the fewest independent channels
        _rec("recurrence long prompt bf16", "forward", "bf16", 1, 65521, 2048, s0=True, view=True),
        # ragged prompts packed into one call, into the cache's slots
        _rec("recurrence packed prompts bf16", "prefill", "bf16", 10, 16384, 2048, s0=True),
        # one user decoding, few key heads
        _heads("heads decode one request", "decode", "bf16", 1, 1, 32, 8, 128, 128, "rms", True),
        # a full batch decoding, every request at its own position
        _heads("heads decode full batch", "decode", "bf16", 256, 1, 32, 32, 128, 128, view=True),
        # prompts on their way into the delta rule: unit keys and queries
        _heads("heads prompts bf16", "forward", "bf16", 4, 4096, 16, 16, 128, 128, view=True),
        # a training step with weighted norms
        _heads("heads train bf16", "train", "bf16", 4, 4096, 32, 8, 128, 128, "rms", True),
        # fp32 training over ragged sizes, part of each head rotated, neighbouring pairs
        _heads("heads train fp32 ragged", "train", "fp32", 3, 1003, 6, 6, 80, 40, "rms", True, True),
    ]


def draw(rng):
    """One more case of the same ranges: sizes spread over their logarithm, odd ones among them,
    at most as many elements as the listed training steps."""

    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("forward", "train", "train", "prefill", "decode"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    if rng.random() < 0.5:
        gate = "fp32" if dtype == "fp32" else rng.choice(("bf16", "fp32"))
        C = log_int(32, 8192)
        if rng.random() < 0.7:  # most layers are multiples of 64 wide, some are odd
            C = max(64, C // 64 * 64)
        if kind == "decode":
            B, T = log_int(1, 256), 1
        elif kind == "prefill":
            B = log_int(2, 80)
            T = log_int(2 * B, min(1 << 16, (1 << 25) // C))
        else:
            B = rng.choice((1, 1, 2, 3, 4, 8))
            T = log_int(1, min(1 << 16, (1 << 25) // (B * C)))
        c = _rec("", kind, dtype, B, T, C, gate, kind in ("prefill", "decode") or rng.random() < 0.5,
                 kind == "forward" and rng.random() < 0.5)
    else:
        D = rng.choice((32, 64, 80, 96, 128, 128, 192, 256, 33))
        R = rng.choice((0, D, D, D // 2)) // 2 * 2
        Hk = rng.choice((1, 2, 3, 4, 8, 16))
        Hq = Hk * rng.choice((1, 1, 2, 4))
        if kind == "decode":
            B, T = log_int(1, 256), 1
        elif kind == "prefill":
            B = log_int(2, 80)
            T = log_int(2 * B, min(1 << 16, (1 << 24) // ((Hq + Hk) * D)))
        else:
            B = rng.choice((1, 1, 2, 3, 4))
            T = log_int(1, min(1 << 15, (1 << 24) // (B * (Hq + Hk) * D)))
        c = _heads("", kind, dtype, B, T, Hq, Hk, D, R, rng.choice(("l2", "rms")), rng.random() < 0.5,
                   rng.random() < 0.3, kind != "train" and rng.random() < 0.5)
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


def _recurrence_inputs(case, seed):
    B, T, C = case["B"], case["T"], case["C"]
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    lead = {"prefill": (1, T), "decode": (B,)}.get(case["kind"], (B, T))
    rate = torch.exp(torch.rand(C, generator=gen, device="cuda") * math.log(1000.0)) * 1e-3
    g = -2.0 * rate * torch.sigmoid(torch.randn(*lead, C, generator=gen, device="cuda"))
    x = torch.randn(*lead, C, generator=gen, device="cuda") * torch.sqrt(-torch.expm1(2.0 * g))
    x, g = x.to(_TYPES[case["dtype"]]), g.to(_TYPES[case["gate"]])
    if case["view"] and x.dtype == g.dtype:
        x, g = torch.cat([x, g], -1).split(C, -1)
    st = {"x": x, "g": g, "s0": None, "cu": None, "slots": None, "gh": None, "gs": None}
    if case["s0"]:
        st["s0"] = torch.randn(B, C, generator=gen, device="cuda")
    if case["kind"] == "prefill":
        st["cu"] = torch.from_numpy(_lengths(case, seed).astype(np.int32)).cuda()
    if case["kind"] in ("prefill", "decode"):
        # a pool half as large again as the batch, which sits on a random part of its slots
        n = B + B // 2 + 1
        st["slots"] = torch.from_numpy(np.sort(np.random.default_rng(seed).permutation(n)[:B]).astype(np.int32)).cuda()
    if case["kind"] == "train":
        st["gh"] = torch.randn(B, T, C, generator=gen, device="cuda").to(_TYPES[case["dtype"]])
        st["gs"] = torch.randn(B, C, generator=gen, device="cuda")
    return st


def _positions(case, seed):
    """Each token's position: prompts from 0, decoding requests anywhere in their context."""
    if case["kind"] == "decode":
        return torch.from_numpy(np.random.default_rng(seed).integers(0, 32768, case["B"]).astype(np.int32)).cuda()
    if case["kind"] == "prefill":
        cu = _lengths(case, seed)
        return torch.from_numpy((np.arange(case["T"]) - np.repeat(cu[:-1], np.diff(cu))).astype(np.int32)).cuda()
    return None  # 0, 1, 2, ... in every row of the batch


def _table(n, R):
    """The rotation's cosines and sines, (n, R): R / 2 cosines, then R / 2 sines."""
    angle = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * torch.exp(
        torch.arange(0, R, 2, device="cuda", dtype=torch.float64) * (-math.log(10000.0) / R))
    return torch.cat([torch.cos(angle), torch.sin(angle)], 1).float()


def _heads_inputs(case, seed):
    B, T, Hq, Hk, D, R = (case[n] for n in ("B", "T", "Hq", "Hk", "D", "R"))
    dt = _TYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    lead = {"prefill": (T,), "decode": (B,)}.get(case["kind"], (B, T))

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["view"]:  # queries, keys and values of one projection
        qkv = normal(*lead, Hq + 2 * Hk, D).to(dt)
        q, k = qkv[..., :Hq, :], qkv[..., Hq:Hq + Hk, :]
    else:
        q, k = normal(*lead, Hq, D).to(dt), normal(*lead, Hk, D).to(dt)
    st = {"q": q, "k": k, "wq": None, "wk": None, "table": None, "pos": None, "gq": None, "gk": None}
    if case["weight"]:
        st["wq"], st["wk"] = 1.0 + 0.1 * normal(D), 1.0 + 0.1 * normal(D)
    if R:
        st["pos"] = _positions(case, seed)
        st["table"] = _table(32768 if case["kind"] == "decode" else T, R)
    if case["kind"] == "train":
        st["gq"], st["gk"] = normal(*lead, Hq, D).to(dt), normal(*lead, Hk, D).to(dt)
    return st


def prepare(case, seed):
    st = {"case": case, **(_recurrence_inputs if case["op"] == "recurrence" else _heads_inputs)(case, seed)}
    if st.get("slots") is not None:
        n = case["B"] + case["B"] // 2 + 1
        if own:
            from prometheus_amd import serving
            st["cache"] = serving.RecurrenceStateCache(1, n, case["C"])
            st["pool"] = st["cache"].pool[0]
        else:
            st["pool"] = torch.zeros(n, case["C"], device="cuda")
        st["pool"][st["slots"].long()] = st["s0"]
    if own and case["kind"] == "train":
        for n in ("x", "g", "s0", "q", "k", "wq", "wk"):
            if st.get(n) is not None:
                st[n].requires_grad_(True)
    return st


# ---------------------------------------------------------------- the plain forms


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1 from zero, by doubling spans."""
    s = 1
    while s < b.shape[1]:
        b = torch.cat([b[:, :s], b[:, s:] + a[:, s:] * b[:, :-s]], 1)
        a = torch.cat([a[:, :s], a[:, s:] * a[:, :-s]], 1)
        s *= 2
    return b


def _plain_recurrence(st):
    case, dt = st["case"], st["x"].dtype
    x, a = st["x"].float(), torch.exp(st["g"].float())
    if case["kind"] == "decode":
        slots = st["slots"].long()
        h = a * st["pool"][slots] + x
        st["pool"][slots] = h
        return {"h": h.to(dt), "pool": st["pool"]}
    if case["kind"] == "prefill":
        slots, cu = st["slots"].long(), st["cu"].long()
        first, full = cu[:-1], cu[1:] > cu[:-1]
        s0 = st["pool"][slots]
        b, keep = x[0].clone(), a[0].clone()
        b[first[full]] += keep[first[full]] * s0[full]
        keep[first[full]] = 0.0  # the state starts anew at every prompt
        h = _scan(keep[None], b[None])
        st["pool"][slots[full]] = h[0, cu[1:][full] - 1]
        return {"h": h.to(dt), "pool": st["pool"]}
    s0 = torch.zeros_like(x[:, 0]) if st["s0"] is None else st["s0"]
    b = x.clone()
    b[:, 0] += a[:, 0] * s0
    h = _scan(a, b)
    out = {"h": h.to(dt), "state": h[:, -1].clone()}
    if case["kind"] == "train":
        # d_t = gh_t + a_{t+1} d_{t+1}: the same scan from the last token to the first
        gh = st["gh"].float().flip(1)
        gh[:, 0] += st["gs"]
        nxt = torch.cat([torch.zeros_like(a[:, :1]), a[:, 1:].flip(1)], 1)
        d = _scan(nxt, gh).flip(1)
        before = torch.cat([s0[:, None], h[:, :-1]], 1)
        out["dx"], out["dg"] = d.to(dt), (d * a * before).to(st["g"].dtype)
        if st["s0"] is not None:
            out["ds0"] = a[:, 0] * d[:, 0]
    return out


def _turn(y, cos, sin, interleaved):
    """Each pair of the first R dimensions turned by its angle; the others stay."""
    half = cos.shape[-1]
    r, rest = y[..., :2 * half], y[..., 2 * half:]
    if interleaved:
        y1, y2 = r[..., 0::2], r[..., 1::2]
        r = torch.stack([y1 * cos - y2 * sin, y2 * cos + y1 * sin], -1).flatten(-2)
    else:
        y1, y2 = r[..., :half], r[..., half:]
        r = torch.cat([y1 * cos - y2 * sin, y2 * cos + y1 * sin], -1)
    return torch.cat([r, rest], -1)


def _plain_heads(st):
    case = st["case"]
    cos = sin = None
    if st["table"] is not None:
        pos = torch.arange(case["T"], device="cuda") if st["pos"] is None else st["pos"].long()
        rows = st["table"][pos]
        half = case["R"] // 2
        cos, sin = rows[..., None, :half], rows[..., None, half:]
    out = {}
    for n in ("q", "k"):
        x, w, gz = st[n].float(), st["w" + n], st["g" + n]
        if case["norm"] == "l2":
            norm = torch.sqrt((x * x).sum(-1, keepdim=True))
            r = 1.0 / norm.clamp_min(1e-6)
        else:
            r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        u = x * r
        y = u if w is None else u * w
        out[n] = (y if cos is None else _turn(y, cos, sin, case["interleaved"])).to(st[n].dtype)
        if gz is None:
            continue
        gy = gz.float()
        if cos is not None:
            gy = _turn(gy, cos, -sin, case["interleaved"])
        if w is not None:
            out["dw" + n] = (gy * u).sum((0, 1, 2))
            gy = gy * w
        dot = (gy * u).sum(-1, keepdim=True)
        if case["norm"] == "l2":
            dx = torch.where(norm > 1e-6, gy - u * dot, gy) * r
        else:
            dx = (gy - u * dot / case["D"]) * r
        out["d" + n] = dx.to(st[n].dtype)
    return out


# ---------------------------------------------------------------- one pass


def _own_recurrence(st):
    from prometheus_amd import kernels
    case, dt = st["case"], st["x"].dtype
    if case["kind"] == "decode":
        return {"h": st["cache"].decode(0, st["slots"], st["x"], st["g"], out_dtype=dt), "pool": st["pool"]}
    if case["kind"] == "prefill":
        h = st["cache"].prefill(0, st["slots"], st["x"], st["g"], st["cu"], out_dtype=dt)
        return {"h": h, "pool": st["pool"]}
    h, s = kernels.linear_recurrence(st["x"], st["g"], st["s0"], out_dtype=dt)
    out = {"h": h.detach(), "state": s.detach()}
    if case["kind"] == "train":
        names = [n for n in ("x", "g", "s0") if st[n] is not None]
        grads = torch.autograd.grad((h, s), [st[n] for n in names], (st["gh"], st["gs"]))
        out.update({"d" + n: g for n, g in zip(names, grads)})
    return out


def _own_heads(st):
    from prometheus_amd import kernels
    case = st["case"]
    q, k = kernels.norm_rotate(st["q"], st["k"], st["table"], st["pos"], norm=case["norm"], q_weight=st["wq"],
                               k_weight=st["wk"], interleaved=case["interleaved"])
    out = {"q": q.detach(), "k": k.detach()}
    if case["kind"] == "train":
        names = [n for n in ("q", "k", "wq", "wk") if st[n] is not None]
        grads = torch.autograd.grad((q, k), [st[n] for n in names], (st["gq"], st["gk"]))
        out.update({"d" + n: g for n, g in zip(names, grads)})
    return out


def run(st):
    if st["case"]["op"] == "recurrence":
        return (_own_recurrence if own else _plain_recurrence)(st)
    return (_own_heads if own else _plain_heads)(st)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    """The forward's inputs read once and its outputs written once; a training pass adds the
    same of the backward, a call of its own that comes after the rest of the model has run."""
    e = 2 if case["dtype"] == "bf16" else 4
    tokens = case["T"] if case["kind"] == "prefill" else case["B"] * case["T"]
    if case["op"] == "recurrence":
        eg = 2 if case["gate"] == "bf16" else 4
        n, states = tokens * case["C"], case["B"] * case["C"] * 4
        nbytes = n * (2 * e + eg) + states * (2 if case["s0"] else 1)
        flops = 3.0 * n
        if case["kind"] == "train":  # x, g, gh in; gx and gg out
            nbytes += n * (3 * e + 2 * eg) + states * (3 if case["s0"] else 1)
            flops += 7.0 * n
        return {"bytes": nbytes, "flops": flops}
    n = tokens * (case["Hq"] + case["Hk"]) * case["D"]
    # the rows of the rotation's table that the positions name, and the positions
    rows = case["B"] if case["kind"] == "decode" else min(case["T"], 32768)
    extra = rows * case["R"] * 4 + (tokens * 4 if case["R"] and case["kind"] in ("decode", "prefill") else 0)
    extra += 8 * case["D"] if case["weight"] else 0
    nbytes, flops = n * 2 * e + extra, 8.0 * n
    if case["kind"] == "train":  # q, k and their outputs' gradients in, gradients out
        nbytes += n * 3 * e + extra + (8 * case["D"] if case["weight"] else 0)
        flops += 16.0 * n
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------- the same in 64 bits


def _walk(x, g, s, out):
    """Token by token: out_t = exp(g_t) out_{t-1} + x_t from s; arrays (N, T, C)."""
    for t in range(x.shape[1]):
        s = torch.addcmul(x[:, t].double(), torch.exp(g[:, t].double()), s, out=out[:, t])
    return s


def _exact_recurrence(case, seed):
    st = _recurrence_inputs(case, seed)
    x, g, f64 = st["x"], st["g"], torch.float64
    if case["kind"] in ("decode", "prefill"):
        slots = st["slots"].long()
        pool = torch.zeros(case["B"] + case["B"] // 2 + 1, case["C"], device="cuda", dtype=f64)
        pool[slots] = st["s0"].double()
        if case["kind"] == "decode":
            h = x.double() + torch.exp(g.double()) * pool[slots]
            pool[slots] = h
            return {"h": h, "pool": pool}
        h, cu = torch.empty(x.shape, device="cuda", dtype=f64), st["cu"].tolist()
        for i, (a, z) in enumerate(zip(cu[:-1], cu[1:])):
            pool[slots[i]] = _walk(x[:, a:z], g[:, a:z], pool[slots[i]][None], h[:, a:z])[0]
        return {"h": h, "pool": pool}
    B, T, C = x.shape
    s0 = torch.zeros(B, C, device="cuda", dtype=f64) if st["s0"] is None else st["s0"].double()
    h = torch.empty(x.shape, device="cuda", dtype=f64)
    state = _walk(x, g, s0, h).clone()
    out = {"h": h, "state": state}
    if case["kind"] == "train":
        out["dx"], out["dg"] = torch.empty_like(h), torch.empty_like(h)
        carry = st["gs"].double()
        for t in range(T - 1, -1, -1):
            d = out["dx"][:, t]
            torch.add(st["gh"][:, t].double(), carry, out=d)
            carry = torch.exp(g[:, t].double()) * d
            torch.mul(carry, h[:, t - 1] if t else s0, out=out["dg"][:, t])
        if st["s0"] is not None:
            out["ds0"] = carry
    return out


def _exact_heads(case, seed):
    st = _heads_inputs(case, seed)
    lead = st["q"].shape[:-2]
    if case["R"]:
        # as complex numbers: a pair is one number, its rotation one product
        pos = st["pos"]
        pos = torch.arange(case["T"], device="cuda").expand(lead) if pos is None else pos.long()
        half = case["R"] // 2
        turn = torch.complex(*(st["table"].double()[pos][..., s][..., None, :]
                               for s in (slice(0, half), slice(half, None))))

    def operator(x, w):
        size = torch.linalg.vector_norm(x, dim=-1, keepdim=True)
        if case["norm"] == "l2":
            y = x / torch.maximum(size, torch.full_like(size, 1e-6))
        else:
            y = x / torch.sqrt(size.square() / case["D"] + 1e-6)
        if w is not None:
            y = y * w
        if not case["R"]:
            return y
        R = case["R"]
        shape = (R // 2, 2) if case["interleaved"] else (2, R // 2)
        pair = y[..., :R].unflatten(-1, shape)
        if not case["interleaved"]:
            pair = pair.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return torch.cat([z, y[..., R:]], -1)

    out = {}
    for n in ("q", "k"):
        train = case["kind"] == "train"
        x = st[n].double().requires_grad_(train)
        w = None if st["w" + n] is None else st["w" + n].double().requires_grad_(train)
        z = operator(x, w)
        out[n] = z.detach()
        if train:
            leaves = [x] if w is None else [x, w]
            grads = torch.autograd.grad(z, leaves, st["g" + n].double())
            out["d" + n] = grads[0]
            if w is not None:
                out["dw" + n] = grads[1]
    return out


def exact(case, seed):
    return (_exact_recurrence if case["op"] == "recurrence" else _exact_heads)(case, seed)
