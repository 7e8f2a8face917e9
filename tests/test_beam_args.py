"""Checks of beam_select's tensors where no scores are given."""
import pytest
import torch

from janus_amd import ops


def test_select_without_scores():
    eng = ops.ComputeEngine(-1)   # good calls reach the library's device check
    logits, out, idx = torch.zeros(6, 50), torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int32)
    for x in (logits, logits.view(2, 3, 50)):
        with pytest.raises(ops.JanusError, match="device"):
            ops.beam_select(eng, x, None, out, idx, idx)
    for bad in (dict(logits=logits[:5]), dict(logits=logits[:1]), dict(out=out[:1]), dict(out=out.view(8)), dict(logits=logits.double())):
        with pytest.raises(ValueError):
            ops.beam_select(eng, bad.get("logits", logits), None, bad.get("out", out), idx, idx)
