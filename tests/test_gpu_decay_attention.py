"""Linear attention with a decay for each head on the GPU, against the 64-bit form.

Tolerances: an output may be off by half a step of its type (bf16 2^-8, fp32 2^-24, relative to its
value) and by the products' accuracy, relative to the same sums over absolute values. For bf16 inputs
the state and the decayed V lose at most 2^-16 each where they are split in two; for fp32 inputs
2^-24 each in three parts and 2^-24 for the products left out; each of the T tokens' terms is added in
fp32 (2^-24 of the sum so far, and the chunk's sum beside it). So 8 * 2^-16 + T 2^-23, and
(T + 64) 2^-23. What comes out in q's type (o, gq, gk, gv) takes, for bf16 inputs, A and the state
as factors in bf16: half a step, 2^-8, of the term that each is in. The gates' gradients take sums of up to 2 * 8 chunks in and out: 17 times that of the
largest one's absolute sum.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import decay_oracle as ref
from prometheus_amd import kernels, serving

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def inputs(B, T, Hq, H, D, dtype, gate="token", s0=True, seed=0, low=-0.3):
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen)

    q, k, v = normal(B, T, Hq, D).to(dtype), (normal(B, T, H, D) / D**0.5).to(dtype), normal(B, T, H, D).to(dtype)
    g = low * torch.rand(*((B, T, H) if gate == "token" else (H,)), generator=gen)
    return q, k, v, g, normal(B, H, D, D) if s0 else None


def eps_of(dtype, T):
    return 8 * 2.0**-16 + T * 2.0**-23 if dtype == BF16 else (T + 64) * 2.0**-23


def eps_out(dtype, T):
    return eps_of(dtype, T) + (2.0**-8 if dtype == BF16 else 0.0)


def near(got, want, size, eps):
    """|got - want| <= half a step of got's type + eps times the sums' size."""
    rnd = torch.finfo(got.dtype).eps / 2
    off = (got.detach().cpu().double() - want).abs()
    allowed = rnd * want.abs() + eps * size + 1e-37
    assert got.shape == want.shape
    assert bool((off <= allowed).all()), (off / allowed).max().item()


def gpu(*xs):
    return [None if x is None else x.cuda() for x in xs]


def size_of(*xs):
    return [None if x is None else x.abs() for x in xs]


def check_forward(q, k, v, g, s0, scale, o, s):
    eo, es = ref.decay(q, k, v, g, s0, scale)
    mo, ms = ref.decay(*size_of(q, k, v), g, *size_of(s0), abs(scale))
    near(o, eo, mo, eps_out(q.dtype, q.shape[1]))
    near(s, es, ms, eps_of(q.dtype, q.shape[1]))


SHAPES = [
    # B, T, Hq, H, D
    (1, 1, 1, 1, 64),
    (2, 2, 2, 1, 16),
    (1, 63, 1, 1, 128),
    (2, 64, 3, 3, 64),
    (1, 65, 4, 2, 33),
    (2, 130, 2, 2, 80),
    (1, 257, 6, 2, 128),
    (1, 100, 2, 2, 200),
    (1, 70, 1, 1, 256),
    (1, 40, 1, 1, 1),
    (1, 100, 2, 2, 100),
    (2, 90, 2, 2, 12),
    (3, 1100, 2, 1, 64),  # several workgroups along the sequence
    (1, 1555, 4, 2, 128),
    (2, 450, 2, 2, 128),  # short, but few heads
    (8, 700, 33, 33, 16),  # longer, but many
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,Hq,H,D", SHAPES)
@pytest.mark.parametrize("gate,s0", [("token", True), ("head", False)])
def test_forward(B, T, Hq, H, D, dtype, gate, s0):
    x = inputs(B, T, Hq, H, D, dtype, gate, s0, seed=T)
    o, s = kernels.decay_attention(*gpu(*x), scale=0.7)
    assert o.dtype == dtype and s.dtype == F32
    check_forward(*x, 0.7, o, s)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,Hq,H,D", SHAPES)
@pytest.mark.parametrize("gate,s0", [("token", True), ("head", False)])
def test_gradients(B, T, Hq, H, D, dtype, gate, s0):
    x = inputs(B, T, Hq, H, D, dtype, gate, s0, seed=T)
    gen = torch.Generator().manual_seed(T + 1)
    go = torch.randn(x[0].shape, generator=gen).to(dtype)
    gs = torch.randn(B, H, D, D, generator=gen) if s0 else None
    dev = gpu(*x)
    leaves = [t for t in dev if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    o, s = kernels.decay_attention(*dev, scale=0.7)
    if gs is None:
        got = torch.autograd.grad(o, leaves, go.cuda())
    else:
        got = torch.autograd.grad((o, s), leaves, (go.cuda(), gs.cuda()))
    check_forward(*x, 0.7, o, s)
    want = ref.decay_bwd(*x, go, gs, 0.7)
    size = ref.decay_bwd(*size_of(*x[:3]), x[3], *size_of(x[4]), go.abs(), *size_of(gs), 0.7)
    eps = eps_of(dtype, T)
    for i, n in enumerate(("q", "k", "v")):
        assert got[i].dtype == dtype
        near(got[i], want[i], size[i], eps_out(dtype, T))
    if gate == "token":
        largest = size[3].amax(1, keepdim=True).expand_as(size[3])
        near(got[3], want[3], largest, 17 * eps)
    else:
        near(got[3], want[3], size[3], 17 * eps)
    if s0:
        near(got[4], want[4], size[4], eps)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_views_of_a_projection(dtype):
    B, T, Hq, H, D = 2, 77, 4, 2, 64
    q, k, v, g, s0 = inputs(B, T, Hq, H, D, dtype)
    wide = torch.cat([q, k, v], 2).cuda()
    parts = wide.split([Hq, H, H], 2)
    assert not parts[0].is_contiguous()
    o, s = kernels.decay_attention(*parts, g.cuda(), s0.cuda())
    check_forward(q, k, v, g, s0, 1.0, o, s)
    # odd offsets of the elements, batch and heads the other way round, gates of a wider projection
    odd = torch.zeros(B, Hq + 2 * H, T, D + 3, dtype=dtype, device="cuda")
    odd[..., 1:D + 1] = wide.transpose(1, 2)
    parts = [p.transpose(1, 2) for p in odd[..., 1:D + 1].split([Hq, H, H], 1)]
    gates = torch.cat([torch.zeros(B, T, 1), g, torch.zeros(B, T, 2)], 2).cuda()[..., 1:1 + H]
    o2, s2 = kernels.decay_attention(*parts, gates, s0.cuda())
    assert torch.equal(o, o2) and torch.equal(s, s2)


def test_expanded_gates_have_gradients_of_each_token():
    q, k, v, g, _ = inputs(2, 70, 2, 2, 64, F32, gate="head")
    dev = gpu(q, k, v)
    per_token = g.cuda().expand(2, 70, 2)
    (o, s), res = kernels.decay_attention_fwd(*dev, per_token)
    go = torch.ones_like(o)
    gg = kernels.decay_attention_bwd(res, (go, None))[3]
    want = ref.decay_bwd(q, k, v, g.expand(2, 70, 2), None, go.cpu(), None)[3]
    size = ref.decay_bwd(*size_of(q, k, v), g.expand(2, 70, 2), None, go.cpu(), None)[3]
    near(gg, want, size.amax(1, keepdim=True).expand_as(size), 17 * eps_of(F32, 70))
    constant = kernels.decay_attention_bwd(kernels.decay_attention_fwd(*dev, g.cuda())[1], (go, None))[3]
    near(constant, want.sum((0, 1)), size.sum((0, 1)), 17 * eps_of(F32, 70))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("G", [1, 2])
@pytest.mark.parametrize("lengths", [[5, 0, 64, 130, 1], [700, 3], [1]])
def test_packed(lengths, G, dtype):
    H, D = 2, 64
    N, n = sum(lengths), len(lengths)
    q, k, v, g, _ = inputs(1, N, G * H, H, D, dtype, seed=N)
    s0 = torch.randn(n, H, D, D, generator=torch.Generator().manual_seed(3))
    cu = np.concatenate([[0], np.cumsum(lengths)])
    got = kernels.decay_attention_varlen(*gpu(q, k, v, g), cu, s0.cuda())
    on_gpu = torch.from_numpy(cu).cuda()
    again = kernels.decay_attention_varlen(*(x[0].cuda() for x in (q, k, v, g)), on_gpu, s0.cuda())
    kernels.check_varlen()
    assert torch.equal(got[0][0], again[0]) and torch.equal(got[1], again[1])
    for i, (a, z) in enumerate(zip(cu[:-1], cu[1:])):
        o, s = got[0][:, a:z], got[1][i:i + 1]
        if a == z:
            assert torch.equal(s.cpu(), s0[i:i + 1])
            continue
        check_forward(q[:, a:z], k[:, a:z], v[:, a:z], g[:, a:z], s0[i:i + 1], 1.0, o, s)


def test_packed_sequences_stay_apart_under_nan():
    q, k, v, g, _ = inputs(1, 40, 2, 2, 64, BF16)
    v[0, 20:] = float("nan")
    o, s = kernels.decay_attention_varlen(*gpu(q, k, v, g), [0, 20, 40])
    assert torch.isfinite(o[:, :20]).all() and torch.isfinite(s[0]).all()
    assert torch.isnan(o[:, 20:]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [1, 30, 32, 33, 64, 100, 128, 256])
@pytest.mark.parametrize("Hq,H", [(2, 2), (4, 2), (10, 2)])
def test_step(dtype, D, Hq, H):
    q, k, v, g, s0 = inputs(3, 1, Hq, H, D, dtype, seed=D)
    state = s0.cuda()
    o = kernels.decay_attention_step(*(x[:, 0].cuda() for x in (q, k, v, g)), state, scale=0.7)
    eo, es = ref.decay(q, k, v, g, s0, 0.7)
    mo, ms = ref.decay(*size_of(q, k, v), g, s0.abs(), 0.7)
    # fp32: D terms of a product, each added in fp32, the state's own rounding among them
    near(o, eo[:, 0], mo[:, 0], (D + 8) * 2.0**-24)
    near(state, es, ms, 8 * 2.0**-24)


def test_decay_of_extremes():
    """Closed gates start anew, also between open ones; a tiny one behind a large one keeps its value."""
    for dtype in (BF16, F32):
        q, k, v, g, s0 = inputs(1, 150, 2, 2, 64, dtype)
        g[:, 10] = -float("inf")
        g[:, 70] = -1e4
        g[:, 71:] = -1e-3
        o, s = kernels.decay_attention(*gpu(q, k, v, g, s0))
        check_forward(q, k, v, g.clamp_min(-1e4), s0, 1.0, o, s)
        none = torch.zeros_like(g)
        check_forward(q, k, v, none, s0, 1.0, *kernels.decay_attention(*gpu(q, k, v, none, s0)))


def test_out_dtype_and_hosts():
    q, k, v, g, s0 = inputs(1, 33, 2, 2, 64, BF16)
    o, s = kernels.decay_attention(*gpu(q, k, v, g, s0), out_dtype=F32)
    assert o.dtype == F32
    check_forward(q, k, v, g, s0, 1.0, o, s)
    ho, hs = kernels.decay_attention(q, k, v, g, s0, out_dtype="fp32")
    assert ho.device.type == "cpu" and torch.equal(ho, o.cpu()) and torch.equal(hs, s.cpu())
    n = [x.float().numpy() for x in (q, k, v, g, s0)]
    no, ns = kernels.decay_attention(*n)
    assert isinstance(no, np.ndarray) and no.dtype == np.float32
    check_forward(*(torch.from_numpy(x) for x in n), 1.0, torch.from_numpy(no), torch.from_numpy(ns))
    state = n[4].copy()
    kernels.decay_attention_step(*(x[:, 0] for x in n[:4]), state)
    assert not np.array_equal(state, n[4])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Hq,H", [(2, 2), (4, 2)])
def test_cache_serves_as_the_whole_sequence(dtype, Hq, H):
    """Prompts of different lengths into the slots, then token by token, against each whole sequence."""
    D, lengths, more = 64, [70, 1, 600], 5
    cache = serving.DecayStateCache(2, 6, H, D)
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    seqs = [inputs(1, n + more, Hq, H, D, dtype, s0=False, seed=n) for n in lengths]
    packed = [torch.cat([s[i][:, :n] for s, n in zip(seqs, lengths)], 1).cuda() for i in range(4)]
    cu = torch.tensor([0, *lengths], dtype=torch.int32).cumsum(0).int().cuda()
    got = [[part] for part in cache.prefill(1, slots, *packed, cu).split(lengths, 1)]
    for t in range(more):
        now = [torch.cat([s[i][:, n + t] for s, n in zip(seqs, lengths)]).cuda() for i in range(4)]
        o = cache.decode(1, slots, *now)
        for i in range(3):
            got[i].append(o[None, i:i + 1])
    cache.check_slots()
    kernels.check_varlen()
    assert not cache.pool[0].any() and not cache.pool[1, [1, 3, 5]].any()
    for i, (s, n) in enumerate(zip(seqs, lengths)):
        check_forward(*s, 1.0, torch.cat(got[i], 1), cache.pool[1, slots[i].long()][None])
    # fixed lengths, from the states that are there
    q, k, v, g, _ = inputs(2, 9, Hq, H, D, dtype, s0=False, seed=1)
    before = cache.pool[1, [2, 0]].cpu()
    o = cache.prefill(1, [2, 0], *gpu(q, k, v, g))
    check_forward(q, k, v, g, before, 1.0, o, cache.pool[1, [2, 0]])


def test_cache_slots_out_of_range():
    cache = serving.DecayStateCache(1, 2, 2, 32)
    cache.pool[:] = 1.0
    q, k, v, g, _ = inputs(3, 6, 2, 2, 32, BF16, s0=False)
    slots = torch.tensor([7, 1, -1], device="cuda")
    o = cache.prefill(0, slots, *gpu(q, k, v, g))
    with pytest.raises(ValueError, match="outside"):
        cache.check_slots()
    s0 = torch.zeros(3, 2, 32, 32)
    s0[1] = 1.0
    want, _ = kernels.decay_attention(*gpu(q, k, v, g, s0))
    assert torch.equal(o, want) and bool((cache.pool[0, 0] == 1.0).all())
    o = cache.decode(0, slots.int(), *(x[:, 0].cuda() for x in (q, k, v, g)))
    assert not o[0].any() and not o[2].any() and bool((cache.pool[0, 0] == 1.0).all())


def test_shared_states_in_place():
    """A group of query heads and several workgroups along the sequence, all from a state that one of
    them replaces."""
    q, k, v, g, s0 = inputs(1, 1300, 4, 1, 64, BF16)
    cache = serving.DecayStateCache(1, 1, 1, 64)
    cache.pool[0] = s0.cuda()
    o = cache.prefill(0, [0], *gpu(q, k, v, g))
    want, s = kernels.decay_attention(*gpu(q, k, v, g, s0))
    assert torch.equal(o, want) and torch.equal(cache.pool[0], s)


def test_graph_replays():
    """A captured decode, prefill and training step, replayed beside eager work."""
    q, k, v, g, s0 = inputs(2, 90, 2, 2, 64, BF16)
    dev = gpu(q, k, v, g, s0)
    go = torch.randn(o_shape := q.shape, device="cuda").to(BF16)

    def step():
        (o, s), res = kernels.decay_attention_fwd(*dev)
        return o, s, *kernels.decay_attention_bwd(res, (go, s))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        fresh = inputs(2, 90, 2, 2, 64, BF16, seed=10 + i)
        for a, b in zip(dev, fresh):
            a.copy_(b)
        go.copy_(torch.randn(o_shape))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)


def test_another_stream():
    x = gpu(*inputs(1, 300, 2, 2, 128, BF16))
    want = kernels.decay_attention(*x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernels.decay_attention(*x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_empty():
    q, k, v, g, s0 = inputs(2, 0, 2, 2, 32, F32)
    dev = gpu(q, k, v, g, s0)
    o, s = kernels.decay_attention(*dev)
    assert o.shape == (2, 0, 2, 32) and torch.equal(s, dev[4])
    (_, _), res = kernels.decay_attention_fwd(*dev)
    gs = torch.randn_like(dev[4])
    grads = kernels.decay_attention_bwd(res, (None, gs))
    assert torch.equal(grads[4], gs) and grads[3].shape == (2, 0, 2)
    none = [x[:0] for x in dev]
    o, s = kernels.decay_attention(*none)
    assert o.shape == (0, 0, 2, 32) and s.shape == (0, 2, 32, 32)
    q, k, v, g, _ = inputs(0, 5, 2, 2, 32, F32, gate="head", s0=False)
    (_, _), res = kernels.decay_attention_fwd(*gpu(q, k, v, g))
    assert not kernels.decay_attention_bwd(res, (None, None))[3].any()


def test_a_missing_gradient():
    q, k, v, g, s0 = inputs(1, 66, 2, 1, 64, F32)
    (o, s), res = kernels.decay_attention_fwd(*gpu(q, k, v, g, s0))
    gs = torch.randn(s.shape).cuda()
    only = kernels.decay_attention_bwd(res, (None, gs))
    both = kernels.decay_attention_bwd(res, (torch.zeros_like(o), gs))
    for a, b in zip(only, both):
        assert torch.equal(a, b)
    assert not only[0].any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_heads_of_a_group_one_after_another(dtype):
    """So much work that a workgroup takes all query heads of a group."""
    x = inputs(64, 800, 8, 4, 16, dtype, seed=5)
    gen = torch.Generator().manual_seed(6)
    go, gs = torch.randn(x[0].shape, generator=gen).to(dtype), torch.randn(64, 4, 16, 16, generator=gen)
    dev = [t.requires_grad_(True) for t in gpu(*x)]
    o, s = kernels.decay_attention(*dev)
    check_forward(*x, 1.0, o, s)
    got = torch.autograd.grad((o, s), dev, (go.cuda(), gs.cuda()))
    want = ref.decay_bwd(*x, go, gs)
    size = ref.decay_bwd(*size_of(*x[:3]), x[3], x[4].abs(), go.abs(), gs.abs())
    for i in range(3):
        near(got[i], want[i], size[i], eps_out(dtype, 800))
    near(got[3], want[3], size[3].amax(1, keepdim=True).expand_as(size[3]), 17 * eps_of(dtype, 800))
    near(got[4], want[4], size[4], eps_of(dtype, 800))


@pytest.mark.parametrize("T", [70, 700])
def test_gradients_without_the_gates(T):
    """Constant decays that are not learned: the same gradients of everything else."""
    q, k, v, g, s0 = inputs(1, T, 2, 1, 64, BF16, gate="head")
    go = torch.randn(q.shape, device="cuda").to(BF16)
    grads = []
    for learned in (True, False):
        dev = gpu(q, k, v, g, s0)
        leaves = [t for i, t in enumerate(dev) if learned or i != 3]
        for t in leaves:
            t.requires_grad_(True)
        got = list(torch.autograd.grad(kernels.decay_attention(*dev)[0], leaves, go))
        if learned:
            del got[3]
        grads.append(got)
    want = ref.decay_bwd(q, k, v, g, s0, go.cpu(), None)
    size = ref.decay_bwd(*size_of(q, k, v), g, s0.abs(), go.cpu().abs(), None)
    for got in grads:
        for i, j in enumerate((0, 1, 2, 4)):
            near(got[i], want[j], size[j], eps_out(BF16, T) if j < 3 else eps_of(BF16, T))


def test_the_first_state_alone_needs_no_gradient():
    """The gates' gradient takes the first state's, also where nobody asks for that."""
    q, k, v, g, s0 = inputs(1, 70, 2, 2, 64, BF16)
    go = torch.randn(q.shape, device="cuda").to(BF16)
    dev = gpu(q, k, v, g, s0)
    dev[3].requires_grad_(True)
    alone, = torch.autograd.grad(kernels.decay_attention(*dev)[0], dev[3:4], go)
    dev[4].requires_grad_(True)
    both = torch.autograd.grad(kernels.decay_attention(*dev)[0], dev[3:5], go)
    assert torch.equal(alone, both[0])


def test_an_fp32_output_of_bf16_inputs():
    q, k, v, g, s0 = inputs(1, 80, 2, 2, 64, BF16)
    dev = [t.requires_grad_(True) for t in gpu(q, k, v, g, s0)]
    o, s = kernels.decay_attention(*dev, out_dtype=F32)
    go = torch.randn(o.shape, device="cuda")
    got = torch.autograd.grad(o, dev, go)
    rounded = torch.autograd.grad(kernels.decay_attention(*dev)[0], dev, go.to(BF16))
    assert all(torch.equal(a, b) for a, b in zip(got, rounded))


def test_saved_tensors_may_come_back_elsewhere():
    """Hooks that park what autograd keeps on the host, in another layout."""
    q, k, v, g, s0 = inputs(1, 70, 4, 2, 64, BF16)

    def grads(pack, unpack):
        dev = [t.requires_grad_(True) for t in gpu(q, k, v, g, s0)]
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            o, s = kernels.decay_attention(*dev)
        return torch.autograd.grad((o, s), dev, (torch.ones_like(o), torch.ones_like(s)))

    want = grads(lambda t: t, lambda t: t)
    for unpack in (lambda t: t, lambda t: t.cuda().transpose(0, -1).contiguous().transpose(0, -1)):
        got = grads(lambda t: t.cpu(), unpack)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_not_differentiable_twice():
    q, k, v, g, s0 = inputs(1, 8, 2, 2, 32, F32)
    dev = [t.requires_grad_(True) for t in gpu(q, k, v, g, s0)]
    o, _ = kernels.decay_attention(*dev)
    gq, = torch.autograd.grad(o.sum(), dev[:1], create_graph=True)
    with pytest.raises(RuntimeError):
        gq.sum().backward()


def test_a_backward_again():
    q, k, v, g, s0 = inputs(1, 600, 2, 2, 64, BF16)
    dev = [t.requires_grad_(True) for t in gpu(q, k, v, g, s0)]
    o, _ = kernels.decay_attention(*dev)
    go = torch.randn(o.shape, device="cuda").to(BF16)
    first = torch.autograd.grad(o, dev, go, retain_graph=True)
    again = torch.autograd.grad(o, dev, go)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("n", [300, 1500])
def test_many_packed_sequences(n):
    """More sequences than threads that count them, most short, some empty, one long."""
    rng = np.random.default_rng(n)
    lengths = rng.integers(0, 6, n)
    lengths[n // 3] = 900
    N, H, D = int(lengths.sum()), 1, 32
    q, k, v, g, _ = inputs(1, N, 1, H, D, BF16, seed=n)
    cu = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)])).cuda()
    o, s = kernels.decay_attention_varlen(*gpu(q, k, v, g), cu)
    kernels.check_varlen()
    a = 0
    for i, length in enumerate(lengths.tolist()):
        if i % 37 == 0 or i == n // 3 or i == n - 1:
            part = [x[:, a:a + length] for x in (q, k, v, g)]
            if length:
                check_forward(*part, None, 1.0, o[:, a:a + length], s[i:i + 1])
            else:
                assert not s[i].any()
        a += length


def test_malformed_offsets_are_reported():
    q, k, v, g, _ = inputs(1, 40, 1, 1, 32, BF16)
    dev = gpu(q, k, v, g)
    kernels.check_varlen()
    for bad in ([0, 50, 40], [0, 30, 20, 40], [-3, 40], [0, 39], [0, 2**33, 40]):
        kernels.decay_attention_varlen(*dev, torch.tensor(bad, device="cuda"))
        with pytest.raises(kernels.KernelError):
            kernels.check_varlen()
    kernels.decay_attention_varlen(*dev, torch.tensor([0, 40], device="cuda"))
    kernels.check_varlen()
    # so many overlapping spans that the slots for them run out
    dev = gpu(*inputs(1, 2000, 1, 1, 32, BF16)[:4])
    kernels.decay_attention_varlen(*dev, torch.tensor([0, 2000] * 9 + [2000], device="cuda"))
    with pytest.raises(kernels.KernelError):
        kernels.check_varlen()


def test_steps_of_views_and_padding():
    q, k, v, g, s0 = inputs(4, 1, 4, 2, 64, BF16)
    wide = torch.cat([q, k, v], 2)[:, 0].cuda()
    state = s0.cuda()
    want = kernels.decay_attention_step(*(x[:, 0].cuda() for x in (q, k, v, g)), state)
    again = s0.cuda()
    gates = torch.cat([torch.zeros(4, 3), g[:, 0]], 1).cuda()[:, 3:]
    got = kernels.decay_attention_step(*wide.split([4, 2, 2], 1), gates, again)
    assert torch.equal(got, want) and torch.equal(again, state)
    cache = serving.DecayStateCache(1, 4, 2, 64)
    cache.pool[0] = s0.cuda()
    slots = torch.tensor([2, -1, 0, 4], dtype=torch.int32, device="cuda")
    out = torch.full((4, 4, 64), 7.0, device="cuda")
    cache.decode(0, slots, *wide.split([4, 2, 2], 1), gates, out)
    assert not out[1].any() and not out[3].any()
    assert torch.equal(cache.pool[0, [1, 3]].cpu(), s0[[1, 3]])


def test_serving_in_a_graph():
    """A captured prefill and decode with slots and offsets that change between replays."""
    H, D, n = 2, 64, 3
    q, k, v, g, _ = inputs(1, 700, 4, H, D, BF16, s0=False)
    dev = gpu(q, k, v, g)
    now = [x[0, :n].contiguous() for x in dev]
    slots = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 100, 600, 700], dtype=torch.int32, device="cuda")
    cache, eager = serving.DecayStateCache(1, 5, H, D), serving.DecayStateCache(1, 5, H, D)
    out = torch.empty_like(now[0])

    def serve(c, out):
        o = c.prefill(0, slots, *dev, cu)
        return o, c.decode(0, slots, *now, out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        serve(cache, out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, _ = serve(cache, out)
    for i, (s, c) in enumerate((([4, 1, 0], [0, 1, 2, 700]), ([2, 3, 1], [0, 0, 650, 700]), ([0, 9, 4], [0, 300, 500, 700]))):
        slots.copy_(torch.tensor(s))
        cu.copy_(torch.tensor(c))
        eager.pool.copy_(cache.pool)
        graph.replay()
        want = serve(eager, torch.empty_like(out))
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(out, want[1]) and torch.equal(cache.pool, eager.pool)


def test_infinities_and_nan_stay_in_their_heads_and_rows():
    q, k, v, g, s0 = inputs(2, 70, 2, 2, 64, BF16)
    v[0, 10, 1] = float("inf")
    q[1, 60, 0] = float("nan")
    o, s = kernels.decay_attention(*gpu(q, k, v, g, s0))
    assert torch.isfinite(o[0, :, 0]).all() and torch.isfinite(o[1, :, 1]).all() and torch.isfinite(s[1]).all()
    assert torch.isfinite(s[0, 0]).all() and not torch.isfinite(o[0, 10:, 1]).any() and torch.isnan(o[1, 60, 0]).all()
    near_ones = torch.ones(1, 5, 1, 32, device="cuda")
    o, s = kernels.decay_attention(near_ones, near_ones, near_ones, torch.tensor([[float("nan")]] * 5, device="cuda")[None])
    assert torch.isnan(o).all() and torch.isnan(s).all()


def test_offsets_past_32_bits():
    B, H, D, half = 1, 128, 128, 65536
    T = 2 * half + 1  # 2.1e9 elements a tensor
    q, k, v, go = (torch.empty(B, T, H, D, dtype=BF16, device="cuda").normal_(std=0.1) for _ in range(4))
    g = torch.full((B, T, H), -0.5, device="cuda")
    (o, s), res = kernels.decay_attention_fwd(q, k, v, g)
    gq, gk, gv, gg, _ = kernels.decay_attention_bwd(res, (go, None))
    # the second half by itself, from nothing: what the first leaves is e^-0.5 of itself a token later, below
    # 2^-180 of it after 256
    tail = [x[:, half:] for x in (q, k, v, g)]
    (o2, s2), res2 = kernels.decay_attention_fwd(*tail)
    two = kernels.decay_attention_bwd(res2, (go[:, half:], None))
    (sizes, s_size), res3 = kernels.decay_attention_fwd(*(x.abs() for x in tail[:3]), tail[3], out_dtype=F32)
    size = kernels.decay_attention_bwd(res3, (go[:, half:].abs(), None))
    # either is off by the file's bounds for sums that decay by e^-0.5 a token (256 terms of them count)
    eps = 2 * eps_out(BF16, 256)
    for got, want, m in ((o, o2, sizes), (gq, two[0], size[0]), (gk, two[1], size[1]), (gv, two[2], size[2])):
        a, b, m = (x[:, 256 - T + half:] if x.shape[1] == T - half else x[:, half + 256:] for x in (got, want, m))
        assert bool(((a.float() - b.float()).abs() <= eps * m.float() + 2.0**-7 * b.float().abs() + 1e-30).all())
    assert bool(((s - s2).abs() <= 2 * eps_of(BF16, 256) * s_size + 1e-30).all())
    largest = size[3].abs().amax(1, keepdim=True)
    assert bool(((gg[:, half + 256:] - two[3][:, 256:]).abs() <= 2 * 17 * eps_of(BF16, 512) * largest).all())


def test_slots_past_32_bits():
    H, D, n = 32, 256, 1100  # 2.3e9 elements of states
    cache = serving.DecayStateCache(1, n, H, D)
    small = serving.DecayStateCache(1, 2, H, D)
    x = [torch.randn(1, 1100, H, D, device="cuda").to(BF16) * 0.1 for _ in range(3)]
    g = -torch.rand(1, 1100, H, device="cuda")
    with torch.no_grad():
        for T in (1100, 60):  # (in spans and whole)
            part = [t[:, :T] for t in x]
            assert torch.equal(cache.prefill(0, [n - 1], *part, g[:, :T]), small.prefill(0, [1], *part, g[:, :T]))
        one = [t[:, 0] for t in x]
        far, near_ = (torch.tensor([i], dtype=torch.int32, device="cuda") for i in (n - 1, 1))
        assert torch.equal(cache.decode(0, far, *one, g[:, 0]), small.decode(0, near_, *one, g[:, 0]))
