"""GPU tests of the operators beside the delta rule where their ranges end: the most heads, offsets
and tables that stand for nothing, saved tensors that come back changed, states without bound."""

from __future__ import annotations

import pytest
import torch

from prometheus_amd import kernels

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def test_the_most_heads():
    """2^24 heads of 256: a head's offset inside its token passes 31 bits. The same bits as in calls
    of a few heads, forward and backward."""
    H, D, cut = 2**24 - 1, 256, 2**22
    q = torch.randn(1, H, D, dtype=BF16, device="cuda")
    k = q[:, :1].contiguous()
    (zq, zk), res = kernels.norm_rotate_fwd(q, k)
    gq, gk, _, _ = kernels.norm_rotate_bwd(res, (zq, zk))
    assert torch.equal(zk, zq[:, :1]) and torch.equal(gk, gq[:, :1])
    for a in range(0, H, cut):
        part = q[:, a:a + cut]
        (want, _), res = kernels.norm_rotate_fwd(part, k)
        assert torch.equal(zq[:, a:a + cut], want), a
        assert torch.equal(gq[:, a:a + cut], kernels.norm_rotate_bwd(res, (want, None))[0]), a
