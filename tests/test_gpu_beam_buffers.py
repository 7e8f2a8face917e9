"""Buffers of janus_beam_select that are the same or overlap."""
import pytest
import torch

from janus_amd import _lib, ops
from test_gpu_beam import DEV, _first, _reference

pytestmark = pytest.mark.gpu


def _call(engine, logits, scores, out, parents, tokens, batch, beams, vocab, n):
    status = engine.lib.janus_beam_select(engine.ctx, logits, scores, out, parents, tokens, batch, beams, vocab, n)
    return status, engine.lib.janus_last_error(engine.ctx).decode()


@pytest.mark.parametrize("batch,beams,vocab", [(40, 4, 3000), (3, 5, 20000)])
def test_scores_in_place(engine, batch, beams, vocab):
    """n = beams: the new scores may replace the old ones, step after step."""
    gen = torch.Generator().manual_seed(71)
    scores = -torch.rand(batch, beams, generator=gen)
    dev = scores.to(DEV)
    parents, tokens = (torch.empty(batch, beams, dtype=torch.int32, device=DEV) for _ in range(2))
    for _ in range(3):
        logits = torch.randn(batch * beams, vocab, generator=gen)
        ops.beam_select(engine, logits.to(DEV), dev, dev, parents, tokens)
        want, at = _first(_reference(logits, scores), beams)
        assert torch.equal(parents.cpu().long(), at // vocab) and torch.equal(tokens.cpu().long(), at % vocab)
        scores = dev.cpu()


def test_outputs_that_overlap_are_refused(engine):
    """What one request writes may be what another one has not read yet."""
    batch, beams, vocab, n = 3, 4, 100, 8
    ints = torch.arange(4000, dtype=torch.int32, device=DEV)
    before, at = ints.clone(), ints.data_ptr()
    good = [at + 4 * 2400, *[at + 4 * 100 * i for i in range(4)]]
    scores, res = 4 * batch * beams, 4 * batch * n
    for i, where in ((2, good[1]), (2, good[1] + scores - 4), (2, good[1] - res + 4), (3, good[1]), (4, good[1]), (2, good[0]),
                     (3, good[0] + 4 * batch * beams * vocab - 4), (4, good[0] - res + 4), (3, good[2]), (4, good[2] + res - 4),
                     (4, good[3]), (4, good[3] - res + 4)):
        args = list(good)
        args[i] = where
        status, said = _call(engine, *args, batch, beams, vocab, n)
        assert status == _lib.E_INVALID_ARG and "overlap" in said, (i, where - at)
    # in place with n below and above beams, and n = beams but an element further on
    for k, out in ((3, good[1]), (5, good[1]), (4, good[1] + 4)):
        status, said = _call(engine, good[0], good[1], out, good[3], good[4], batch, beams, vocab, k)
        assert status == _lib.E_INVALID_ARG and "overlap" in said, (k, out - at)
    engine.sync()
    assert torch.equal(ints, before)
    for args in ([good[0], None, *good[1:4]], [good[0], good[1], good[1] + scores, good[1] + scores + res, good[1] + scores + 2 * res]):
        ints[2400:3600] = 0   # logits
        assert _call(engine, *args, batch, beams, vocab, n)[0] == _lib.OK
    engine.sync()


@pytest.mark.parametrize("batch,beams,vocab,n", [(1, 1, 900, 4), (3, 4, 9000, 8)])
def test_without_scores(engine, batch, beams, vocab, n):
    logits = torch.randn(batch, beams, vocab, generator=torch.Generator().manual_seed(72))
    out = torch.empty(batch, n, device=DEV)
    parents, tokens = (torch.empty(batch, n, dtype=torch.int32, device=DEV) for _ in range(2))
    ops.beam_select(engine, logits.to(DEV), None, out, parents, tokens)
    _, at = _first(_reference(logits, torch.zeros(batch, beams)), n)
    assert torch.equal(parents.cpu().long(), at // vocab) and torch.equal(tokens.cpu().long(), at % vocab)
