"""GPU test of examples/hybrid_decoder.py: it learns, and serves what it computes."""

from __future__ import annotations

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "hybrid_decoder.py")


def test_trains_and_serves():
    spec = importlib.util.spec_from_file_location("hybrid_decoder", PATH)
    hybrid = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(hybrid)
    torch.manual_seed(0)
    vocab, layers = 64, 4
    model = hybrid.Hybrid(vocab, 512, layers).cuda()
    losses = hybrid.train(model, 160, 8, 512, vocab, say=lambda *a, **k: None)
    assert torch.isfinite(losses).all()
    # below the logarithm of the vocabulary, which is what knowing nothing costs
    assert losses[-20:].mean() < 0.75 * torch.tensor(float(vocab)).log()
    # Served token by token against whole sequences: the same sums in other orders, rounded to
    # bf16 at some ten places a layer, half a step of 2^-8 each.
    for got, want in hybrid.serve(model, [70, 1, 300, 33], 20, vocab):
        assert got.shape == want.shape
        assert (got - want).abs().max() <= 10 * layers * 2.0**-8 * want.abs().max()
