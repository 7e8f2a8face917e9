"""The sums of exponentials that beams are compared by: scores near their logarithm leave values near 0, whose last bits
show how far the sums are off."""
import math

import pytest
import torch

from janus_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _best(engine, logits, scores):
    out = torch.empty(scores.shape[0], 1, device=DEV)
    parents, tokens = (torch.empty(out.shape, dtype=torch.int32, device=DEV) for _ in range(2))
    ops.beam_select(engine, logits, scores.to(DEV), out, parents, tokens)
    return out.cpu().double(), tokens.cpu()


@pytest.mark.parametrize("vocab", [20_000_001, 33_333_335])
def test_sums_beyond_binary32(engine, vocab):
    """Equal logits: all terms are 1, and their number is no binary32 value, nor are the sums of some of the parts'."""
    assert float(torch.tensor(float(vocab))) != vocab
    score = torch.tensor([[math.log(vocab)]])
    out, tokens = _best(engine, torch.full((1, vocab), -3.0, device=DEV), score)
    want = float(score.double()) - math.log(vocab)
    # the logarithm and the sum with the score in binary64, 2^-52 of 18 a step; the value in binary32
    assert abs(float(out) - want) <= abs(want) * U + 18 * 2.0 ** -50 and int(tokens) == 0


@pytest.mark.parametrize("vocab,sigma", [(515, 1.0), (32000, 3.0), (128256, 0.5), (128256, 3.0)])
def test_values_near_zero(engine, vocab, sigma):
    logits = torch.randn(4, vocab, generator=torch.Generator().manual_seed(vocab)) * sigma
    x = logits.double()
    rest = torch.logsumexp(x, -1) - x.amax(-1)
    scores = rest.float()[:, None]
    out, tokens = _best(engine, logits.to(DEV), scores)
    want = scores.double()[:, 0] - rest
    # a term: the difference t to a maximum is rounded, so is its product with log2(e), twice (3 |t| u in all), and the
    # exponential by a step (2 u); 16 terms are added in binary32 (15 u); all else is in binary64
    t = x.amax(-1, keepdim=True) - x
    tol = ((torch.softmax(x, -1) * t).sum(-1) * 3 + 17) * U + want.abs() * U
    assert ((out[:, 0] - want).abs() <= tol).all(), ((out[:, 0] - want).abs() / tol)
    assert torch.equal(tokens[:, 0].long(), logits.argmax(-1))
