"""CPU tests of decay attention and the norms around it at the edges of their sizes: what they plan or
refuse there, before any device work."""

from __future__ import annotations

import pytest
import torch

from prometheus_amd import _native, kernels, serving
from prometheus_amd.kernels import row_norms

MOST = 2**31 - 1 - 1024  # tokens of a sequence


@pytest.mark.parametrize("H", [1, 8])
def test_workspaces_of_very_many_tokens(H):
    """A sequence of many tokens is cut into spans, whose states the workspace holds, up to the last length
    that a call takes (sums of a length and a span's pass 2^31 from about 2.13e9 on)."""
    L = _native.lib()
    sizes = [
        lambda T: L.pm_decay_attention_workspace_bytes(1, T, H, H, 1, 0, 0),
        lambda T: L.pm_decay_attention_workspace_bytes(1, T, H, H, 1, 1, 0),
        lambda T: L.pm_decay_attention_workspace_bytes(3, T, H, H, 1, 1, 1),
    ]
    if H == 1:  # (more heads would take more workgroups than a launch of the backward has)
        sizes.append(lambda T: L.pm_decay_attention_bwd_workspace_bytes(1, T, H, H, 1, 0))
    lengths = (2_000_000_000, 2_131_000_000, 2_144_000_000, 2_145_500_000, MOST)
    for i, size in enumerate(sizes):
        got = [size(T) for T in lengths]
        # (a state and its log-decay are 12 bytes; the card holds 768 workgroups, three of them to a span of
        # the backward)
        assert min(got) >= 12 * 250, (i, got)
        assert max(got) <= 1.5 * min(got), (i, got)  # (as many spans as the card holds)
        assert size(MOST + 1) == 0


EMPTY = [(0, 16), (2, 0, 16), (0, 5, 16), (2, 0, 4, 16), (3, 0, 2, 5, 8), (2, 3, 0, 16), (0, 0, 8)]


@pytest.mark.parametrize("shape", EMPTY)
def test_no_rows_are_evenly_spaced(shape):
    """Wherever the dimension without elements stands, for contiguous tensors and for views."""
    x = torch.zeros(shape)
    wide = torch.zeros(*shape[:-1], shape[-1] + 3)[..., 1:shape[-1] + 1]
    for a in (x, wide):
        rows, inner, strides = row_norms._rows_of(shape, a.stride(), x.stride())
        assert rows == 0 and inner == 1 and len(strides) == 4
        assert row_norms._even(shape[:-1], a.stride()[:-1]) is not None


@pytest.mark.parametrize("sizes", [(1, 2**32 + 5, 2, 2), (2**32 + 2, 1, 2, 2), (1, 3, 2**32 + 2, 2)])
def test_sizes_past_32_bits_are_refused(sizes):
    """A view may have them without memory; the library's own sizes are 32-bit ones."""
    B, T, Hq, H = sizes
    q, k = torch.zeros(1, 1, 1, 1).expand(B, T, Hq, 1), torch.zeros(1, 1, 1, 1).expand(B, T, H, 1)
    g = torch.zeros(H)
    calls = [lambda: kernels.decay_attention(q, k, k, g), lambda: kernels.decay_attention_fwd(q, k, k, g),
             lambda: serving.DecayStateCache(1, 2, H, 1, device="cpu").prefill(0, [0], q, k, k, g)]
    if max(B, Hq) >= 2**31:
        calls.append(lambda: kernels.decay_attention_step(q[:, 0], k[:, 0], k[:, 0], g,
                                                          torch.zeros(1).expand(B, H, 1, 1)))
    for f in calls:
        with pytest.raises(kernels.KernelError, match="too large"):
            f()


def test_rows_of_more_than_32_bits_are_copied():
    shape = (2, 2**31, 8)
    assert row_norms._rows_of(shape, (2**40, 16, 1), (2**34, 8, 1)) is None
    rows, inner, strides = row_norms._rows_of(shape, (2**35, 16, 1), (2**34, 8, 1))
    assert (rows, inner, list(strides)) == (2**32, 1, [16, 0, 8, 0])


def test_spans_by_the_head_dimension():
    """Sequences are cut (and the workspace holds the states between) where the card holds twice as many
    workgroups, between D 65 and 128 three times as many, and only then."""
    L = _native.lib()

    def states(T, H, D):
        return L.pm_decay_attention_workspace_bytes(1, T, H, H, D, 0, 0) // (4 * H * D * D)

    for D, resident, tiles, more in ((16, 768, 1, 2), (64, 768, 1, 2), (65, 512, 1, 3), (128, 512, 1, 3), (129, 256, 2, 2),
                                     (256, 256, 2, 2)):
        H = resident // (more * tiles)
        assert states(4096, H, D) >= 2 and states(4096, H + 1, D) == 0, D
        assert states(200, 1, D) == 0 and states(400, 1, D) >= 2
