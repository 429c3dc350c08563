"""How near decay attention comes to the 64-bit form: bounds of the error's root mean square, for the GPU
tests and for those on the CPU that plant lost parts of factors.

Errors are counted against the spread, the root of the sum of squares of an output's terms, since the
terms' errors are independent. A sum in fp32 rounds by at most 2^-24 of itself at each addition: over T
tokens, G heads of a group and D elements sqrt(T G + D) 2^-24. The decays' factors are off by 2^-24 once a
chunk of 32 tokens, the same way in all terms: T / 32 of that. A factor in three bf16 parts is off by at
most 2^-24 (five of them at most, and the products left out: 8 in all), one in two parts by 2^-17
(half a step of the second part, which is at most 2^-8 of the value and itself off by 2^-9 of that).
The decays' gradients hand what they sum over up to 16 chunks on from chunk to chunk, each chunk's own
sums once in and once out: sqrt(33) of one's, 6.
What comes out in bf16 is rounded once: the exact value's own rounding error, and 2% for the values that
another rounding falls upon.
"""

import torch

from oracle import decay_oracle as ref

BF16, F32 = torch.bfloat16, torch.float32


def of_sums(T, G, D):
    return (8 + T / 32 + (T * G + D) ** 0.5) * 2.0**-24


def of_factors(dtype, T, G, D):
    """Where the state and A are factors: in two parts next to bf16 inputs."""
    return of_sums(T, G, D) + (2.0**-16 if dtype == BF16 else 0.0)  # (two factors, the state and A)


def bound(want, spread, out_dtype, eps):
    """What the rms of an output's error may be."""
    most = eps * ref.rms(spread)
    if out_dtype == BF16:
        most += 1.02 * ref.rms(want.float().bfloat16().double() - want)
    return most + 1e-37


def check(got, want, spread, eps):
    assert got.shape == want.shape
    off, most = ref.rms(got.detach().cpu().double() - want), bound(want, spread, got.dtype, eps)
    assert off <= most, (off, most)


def inputs(B, T, Hq, H, D, dtype, s0=True, seed=0, low=-0.3, zeros=False):
    """Unit normal values, keys of norm one, log-decays from [low, 0] per token (a third of them 0)."""
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen)

    q, k, v = normal(B, T, Hq, D).to(dtype), (normal(B, T, H, D) / D**0.5).to(dtype), normal(B, T, H, D).to(dtype)
    g = low * torch.rand(B, T, H, generator=gen)
    if zeros:
        g = torch.where(torch.rand(B, T, H, generator=gen) < 1 / 3, 0.0, g)
    go, gs = normal(B, T, Hq, D).to(dtype), normal(B, H, D, D)
    return q, k, v, g, normal(B, H, D, D) if s0 else None, go, gs


def bound_gates(spread, T, G, D):
    """What the rms of the decays' gradient's error may be. What a chunk's tokens add to it or take from it
    are parts of the gradient at the chunk's first token and behind its last; where a span begins it is a
    product of two states, whose sums' errors are handed to all of its tokens. (Factors are in three parts,
    for bf16 inputs too.)"""
    return 6 * of_sums(T, G, D) * ref.rms(spread.amax(1, keepdim=True).expand_as(spread))


def check_gates(got, want, spread, T, G, D):
    assert got.shape == want.shape and got.dtype == F32
    off, most = ref.rms(got.detach().cpu().double() - want), bound_gates(spread, T, G, D)
    assert off <= most, (off, most)


def slow(B, T, Hq, H, D, dtype, seed=0):
    """Inputs whose states live through the whole sequence: rates of 0 to 0.002 a token."""
    return inputs(B, T, Hq, H, D, dtype, seed=seed, low=-2e-3, zeros=True)
