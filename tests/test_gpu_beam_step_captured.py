"""A whole step of beam search over a 4-bit cache in one captured graph: append, attention, selection with the scores
in place, reordering by the parents that it wrote; replays against the same step run eagerly."""
import pytest
import torch

from janus_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BATCH, BEAMS, HEADS, KVH, HD, VOCAB, CAP = 3, 4, 8, 2, 128, 5000, 700


class Step:
    def __init__(self, gen):
        rows = BATCH * BEAMS
        self.caches = [torch.zeros(rows * CAP, KVH, HD // d, dtype=torch.uint8, device=DEV) for d in (2, 32, 2, 32)]
        self.base = (torch.randperm(rows, generator=gen) * CAP).int().to(DEV)
        self.head = torch.randn(HEADS * HD, VOCAB, generator=gen).to(DEV) * 0.05
        self.embed = torch.randn(VOCAB, HEADS + 2 * KVH, HD, generator=gen).to(DEV)
        self.pos = torch.full((rows,), 500, dtype=torch.int32, device=DEV)
        self.lens = torch.full((rows,), 501, dtype=torch.int32, device=DEV)
        self.tokens = torch.randint(0, VOCAB, (BATCH, BEAMS), generator=gen, dtype=torch.int32).to(DEV)
        self.parents = torch.zeros(BATCH, BEAMS, dtype=torch.int32, device=DEV)
        self.scores = torch.full((BATCH, BEAMS), -float("inf"), device=DEV)
        self.scores[:, 0] = 0
        self.out = torch.empty(rows, HEADS, HD, device=DEV)
        # a context of 500 positions in every slot
        kv = torch.randn(rows * 500, 2, KVH, HD, generator=gen).to(DEV)
        at = torch.arange(500, dtype=torch.int32, device=DEV).repeat(rows)
        self.context = (kv, self.base.repeat_interleave(500).contiguous(), at)

    def fill(self, e):
        kv, base, at = self.context
        ops.kv_update_fp4(e, kv[:, 0], kv[:, 1], *self.caches, CAP, row_base=base, positions=at)

    def run(self, e):
        rows = BATCH * BEAMS
        x = self.embed[self.tokens.view(-1).long()].contiguous()
        ops.kv_update_fp4(e, x[:, HEADS:HEADS + KVH], x[:, HEADS + KVH:], *self.caches, CAP, row_base=self.base, positions=self.pos)
        q = x[:, :HEADS].contiguous()
        ops.fp4_attention(e, q, *self.caches, self.out, rows, CAP, row_base=self.base, seq_lens=self.lens)
        # the product's order of additions is the same for every run of one shape
        logits = (self.out.view(rows, -1) @ self.head).contiguous()
        ops.beam_select(e, logits, self.scores, self.scores, self.parents, self.tokens)
        ops.kv_reorder(e, self.caches, BEAMS, CAP, self.base, self.parents, seq_lens=self.lens)
        self.pos += 1
        self.lens += 1

    def state(self):
        return [*self.caches, self.pos, self.lens, self.tokens, self.parents, self.scores, self.out]


def test_a_captured_step_is_the_eager_one(engine):
    one, two = (Step(torch.Generator().manual_seed(81)) for _ in range(2))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        engine.bind_stream(stream)
        try:
            for s in (one, two):
                s.fill(engine)
                s.run(engine)
            stream.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                one.run(engine)
            for i in range(6):
                g.replay()
                stream.synchronize()
                two.run(engine)
                stream.synchronize()
                for k, (a, b) in enumerate(zip(one.state(), two.state())):
                    assert torch.equal(a, b), (i, k)
            assert int(two.lens[0]) == 508 and torch.isfinite(two.scores).all()
            assert (two.parents != torch.arange(BEAMS, device=DEV, dtype=torch.int32)).any()
        finally:
            engine.bind_stream(torch.cuda.default_stream())
