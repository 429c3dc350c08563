"""A small hybrid decoder: recurrence layers between delta-rule layers, trained and then served.

    python examples/hybrid_decoder.py [--steps 200] [--layers 4] [--width 512] [--batch 8] [--tokens 512]

Every second layer keeps a vector state (``kernels.linear_recurrence``: its input and log-gate are
the halves of one projection, read in place), the others a matrix state per head
(``kernels.norm_rotate`` on the queries and keys of one projection, then
``kernels.chunked_delta_rule``). The model learns to continue sequences that repeat themselves;
then prompts of different lengths are prefilled in one packed call and continued token by token
from the state caches, and the logits are compared with those of the whole sequences at once.
"""

from __future__ import annotations

import argparse
import os
import sys
import time

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from prometheus_amd import kernels, serving  # noqa: E402

BF16 = torch.bfloat16


def rms(x):
    return F.rms_norm(x.float(), x.shape[-1:]).to(BF16)


class Recurrence(torch.nn.Module):
    """x -> out(silu(z) h) with h the gated linear recurrence of the projection's halves."""

    def __init__(self, width):
        super().__init__()
        self.width = width
        self.proj = torch.nn.Linear(width, 3 * width, bias=False)
        self.out = torch.nn.Linear(width, width, bias=False)
        # memories from the last token to some hundreds
        self.rate = torch.nn.Parameter(torch.linspace(-6.0, 3.0, width))

    def parts(self, x):
        y, g, z = F.linear(rms(x), self.proj.weight.to(BF16)).split(self.width, -1)
        log_gate = -F.softplus(g.float() + self.rate)  # at most 0: the state decays
        # an input of the size that keeps the state of order one
        return y * torch.sqrt(-torch.expm1(2.0 * log_gate)).to(BF16), log_gate, z

    def finish(self, h, z):
        return F.linear(h * F.silu(z), self.out.weight.to(BF16))

    def forward(self, x):
        y, log_gate, z = self.parts(x)
        h, _ = kernels.linear_recurrence(y, log_gate, out_dtype=BF16)
        return self.finish(h, z)

    def prefill(self, x, cache, layer, slots, cu, positions):
        y, log_gate, z = self.parts(x)
        return self.finish(cache.prefill(layer, slots, y, log_gate, cu, out_dtype=BF16), z)

    def decode(self, x, cache, layer, slots, positions):
        y, log_gate, z = self.parts(x)
        return self.finish(cache.decode(layer, slots, y, log_gate, out_dtype=BF16), z)


class DeltaRule(torch.nn.Module):
    """Delta-rule attention with weighted, rotated unit queries and keys."""

    def __init__(self, width, dim, table):
        super().__init__()
        self.heads, self.dim, self.table = width // dim, dim, table
        self.proj = torch.nn.Linear(width, 3 * width, bias=False)
        self.beta = torch.nn.Linear(width, self.heads)
        self.out = torch.nn.Linear(width, width, bias=False)
        self.q_weight = torch.nn.Parameter(torch.ones(dim))

    def parts(self, x, positions):
        x = rms(x)
        qkv = F.linear(x, self.proj.weight.to(BF16)).unflatten(-1, (3 * self.heads, self.dim))
        q, k, v = qkv.split(self.heads, -2)
        # (the delta rule wants unit keys: no weight on k)
        q, k = kernels.norm_rotate(q, k, self.table, positions, q_weight=self.q_weight)
        return q, k, v.contiguous(), torch.sigmoid(self.beta(x.float()))

    def finish(self, o):
        return F.linear(o.to(BF16).flatten(-2), self.out.weight.to(BF16))

    def forward(self, x):
        return self.finish(kernels.chunked_delta_rule(*self.parts(x, None))[0])

    def prefill(self, x, cache, layer, slots, cu, positions):
        q, k, v, beta = (t[None] for t in self.parts(x, positions))
        return self.finish(cache.prefill(layer, slots, q, k, v, beta, cu)[0])

    def decode(self, x, cache, layer, slots, positions):
        return self.finish(cache.decode(layer, slots, *self.parts(x, positions)))


class Hybrid(torch.nn.Module):
    def __init__(self, vocab, width, layers, dim=64, max_tokens=4096):
        super().__init__()
        table = kernels.rotation_table(max_tokens, dim)
        self.width, self.dim = width, dim
        self.embed = torch.nn.Embedding(vocab, width)
        self.head = torch.nn.Linear(width, vocab, bias=False)
        self.layers = torch.nn.ModuleList(
            Recurrence(width) if i % 2 == 0 else DeltaRule(width, dim, table) for i in range(layers))

    def logits(self, x):
        return F.linear(rms(x), self.head.weight.to(BF16)).float()

    def forward(self, tokens):
        x = self.embed(tokens)
        for layer in self.layers:
            x = x + layer(x).float()
        return self.logits(x)

    def caches(self, n_slots):
        """A state cache for each kind of layer, and each layer's place in its own."""
        vectors = [layer for layer in self.layers if isinstance(layer, Recurrence)]
        matrices = [layer for layer in self.layers if isinstance(layer, DeltaRule)]
        kept = {Recurrence: serving.RecurrenceStateCache(len(vectors), n_slots, self.width)}
        if matrices:
            kept[DeltaRule] = serving.LinearStateCache(len(matrices), n_slots, matrices[0].heads, self.dim)
        return [(kept[type(layer)], (vectors if type(layer) is Recurrence else matrices).index(layer))
                for layer in self.layers]

    @torch.no_grad()
    def prefill(self, tokens, cu, slots, caches):
        """Packed prompts (N,): the logits of every token; the states are in the slots."""
        cu_host = cu.tolist()
        positions = torch.cat([torch.arange(z - a) for a, z in zip(cu_host[:-1], cu_host[1:])]).int().cuda()
        x = self.embed(tokens)
        for layer, (cache, at) in zip(self.layers, caches):
            x = x + layer.prefill(x, cache, at, slots, cu, positions).float()
        return self.logits(x)

    @torch.no_grad()
    def decode(self, tokens, positions, slots, caches):
        """One token per request (B,), at its position."""
        x = self.embed(tokens)
        for layer, (cache, at) in zip(self.layers, caches):
            x = x + layer.decode(x, cache, at, slots, positions).float()
        return self.logits(x)


def repeating(batch, tokens, vocab, period, gen):
    """Random sequences that repeat themselves after ``period`` tokens."""
    first = torch.randint(0, vocab, (batch, period), generator=gen, device="cuda")
    return first.repeat(1, -(-tokens // period))[:, :tokens]


def train(model, steps, batch, tokens, vocab, period=32, lr=1e-3, say=print):
    gen = torch.Generator(device="cuda").manual_seed(1)
    opt = torch.optim.AdamW(model.parameters(), lr=lr)
    losses, start = [], None
    for step in range(steps):
        seq = repeating(batch, tokens + 1, vocab, period, gen)
        loss = F.cross_entropy(model(seq[:, :-1])[:, period:].flatten(0, 1), seq[:, period + 1:].flatten())
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if step == 4:
            torch.cuda.synchronize()
            start = time.perf_counter()
        if step % 40 == 0 or step == steps - 1:
            say(f"step {step}: loss {loss.item():.4f}", flush=True)
    if start is not None and steps > 5:
        torch.cuda.synchronize()
        say(f"{(steps - 5) * batch * tokens / (time.perf_counter() - start):.3g} tokens/s", flush=True)
    return torch.stack(losses)


def serve(model, lengths, more, vocab, period=32):
    """Prefills ragged prompts in one call and feeds ``more`` tokens each one by one; returns the
    logits of every request's tokens and those of its whole sequence at once."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    n = len(lengths)
    seqs = [repeating(1, length + more, vocab, period, gen)[0] for length in lengths]
    caches = model.caches(n + 2)
    slots = torch.arange(n, 0, -1, dtype=torch.int32, device="cuda")
    ends = torch.tensor([0, *lengths]).cumsum(0).int().cuda()
    prompts = torch.cat([s[:length] for s, length in zip(seqs, lengths)])
    packed = model.prefill(prompts, ends, slots, caches)
    got = [[part] for part in packed.split(lengths)]
    at = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for t in range(more):
        now = torch.stack([s[length + t] for s, length in zip(seqs, lengths)])
        step = model.decode(now, at + t, slots, caches)
        for i in range(n):
            got[i].append(step[i:i + 1])
    with torch.no_grad():
        return [(torch.cat(parts), model(s[None])[0]) for parts, s in zip(got, seqs)]


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--steps", type=int, default=200)
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--width", type=int, default=512)
    p.add_argument("--batch", type=int, default=8)
    p.add_argument("--tokens", type=int, default=512)
    a = p.parse_args()
    torch.manual_seed(0)
    vocab = 64
    model = Hybrid(vocab, a.width, a.layers).cuda()
    train(model, a.steps, a.batch, a.tokens, vocab)
    for i, (got, want) in enumerate(serve(model, [70, 1, 300, 33], 20, vocab)):
        off = (got - want).abs().max().item() / want.abs().max().item()
        same = (got.argmax(-1) == want.argmax(-1)).float().mean().item()
        print(f"request {i}: {len(got)} tokens, served against whole: largest difference {off:.4f} of the largest "
              f"logit, {100 * same:.1f}% of the choices alike")


if __name__ == "__main__":
    main()
