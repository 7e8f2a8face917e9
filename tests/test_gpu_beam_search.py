"""The operators of the 4-bit cache and of beam search together: prompts, the fork into
beams, decode steps, selection and reordering, layer by layer, against histories kept as
lists on the CPU."""
import numpy as np
import pytest
import torch

from janus_amd import ops
from fp4_ref import decode, encode
from packed_ref import attend, check
from test_gpu_beam import _first, _reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LAYERS, BEAMS, HEADS, KVH, HD, HIDDEN, VOCAB, CAP = 2, 4, 4, 2, 64, 128, 1000, 48


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _weight(engine, rng, n, k, size):
    w = (rng.standard_normal((n, k), dtype=np.float32) * size).astype(np.float16)
    return ops.GpuTensor(engine, ops.DT_F16, n, k, w)


class Search:
    """A small model whose steps call the operators as a server would."""

    def __init__(self, engine, requests):
        rng = np.random.default_rng(7)
        self.engine, self.requests = engine, requests
        self.embedding = torch.from_numpy(rng.standard_normal((VOCAB, HIDDEN), dtype=np.float32)).to(DEV)
        self.qkv = [_weight(engine, rng, (HEADS + 2 * KVH) * HD, HIDDEN, 0.15) for _ in range(LAYERS)]
        self.o = [_weight(engine, rng, HIDDEN, HEADS * HD, 0.05) for _ in range(LAYERS)]
        self.head = _weight(engine, rng, VOCAB, HIDDEN, 0.12)
        self.rope = ops.create_rope_cache(engine, CAP, HD, 10000.0)
        rows = requests * BEAMS * CAP
        self.caches = [torch.zeros(LAYERS, rows, KVH, HD // d, dtype=torch.uint8, device=DEV) for d in (2, 32, 2, 32)]
        # slots in an order of their own
        self.base = [s * CAP for s in np.random.default_rng(8).permutation(requests * BEAMS).tolist()]

    def forward(self, tokens, slots, positions, q_start, lens, trace):
        """One pass of packed rows; row r of sequence s goes to slot slots[s]. Returns the last layer's rows."""
        e, rows = self.engine, len(tokens)
        owner = [s for s, (a, b) in enumerate(zip(q_start[:-1], q_start[1:])) for _ in range(b - a)]
        row_base = _i32([self.base[slots[s]] for s in owner])
        pos = _i32(positions)
        x = self.embedding[torch.tensor(tokens, device=DEV)].contiguous()
        for layer in range(LAYERS):
            qkv = torch.empty(rows, HEADS + 2 * KVH, HD, device=DEV)
            ops.gemm_auto(e, x, self.qkv[layer], qkv, 1, rows, HIDDEN, (HEADS + 2 * KVH) * HD)
            heads = qkv[:, :HEADS + KVH].contiguous()
            ops.rope(e, heads, heads, self.rope, rows, HEADS + KVH, HD, 0, pos)
            q, k, v = heads[:, :HEADS].contiguous(), heads[:, HEADS:], qkv[:, HEADS + KVH:]
            cache = [c[layer] for c in self.caches]
            ops.kv_update_fp4(e, k, v, *cache, CAP, row_base=row_base, positions=pos)
            out = torch.empty_like(q)
            ops.fp4_attention(e, q, *cache, out, len(slots), CAP, q_start=_i32(q_start), seq_lens=_i32(lens),
                              row_base=_i32([self.base[s] for s in slots]))
            trace(layer, q.cpu(), k.cpu(), v.cpu(), out)
            y = torch.empty(rows, HIDDEN, device=DEV)
            ops.gemm_residual(e, out.view(rows, -1), self.o[layer], x, y, rows)
            x = y
        return x

    def logits(self, x):
        out = torch.empty(x.shape[0], VOCAB, device=DEV)
        ops.gemm_auto(self.engine, x.contiguous(), self.head, out, 1, x.shape[0], HIDDEN, VOCAB)
        return out

    def reorder(self, parents, lens):
        ops.kv_reorder(self.engine, self.caches, BEAMS, CAP, _i32(self.base), _i32(parents), seq_lens=_i32(lens), layers=LAYERS)


def _appended(history, rows):
    return torch.cat([history, decode(*encode(rows))])


def test_beam_search_over_a_4_bit_cache(engine):
    prompts = [np.random.default_rng(i).integers(0, VOCAB, n).tolist() for i, n in enumerate((5, 13, 1))]
    requests = len(prompts)
    search = Search(engine, requests)
    empty = torch.zeros(0, KVH, HD, dtype=torch.float64)
    k_of, v_of = ([[empty] * (requests * BEAMS) for _ in range(LAYERS)] for _ in range(2))   # histories of every slot

    def trace_of(slots, q_start):
        def trace(layer, q, k, v, out):
            for s, a, b in zip(slots, q_start[:-1], q_start[1:]):
                k_of[layer][s], v_of[layer][s] = _appended(k_of[layer][s], k[a:b]), _appended(v_of[layer][s], v[a:b])
                n = len(k_of[layer][s])
                want, tol = attend(q[a:b], k_of[layer][s], v_of[layer][s], [n - (b - a) + 1 + i for i in range(b - a)], False, True)
                check(out[a:b], want, tol, (layer, s, n))
        return trace

    # the prompts, packed, into the first slot of each request
    firsts = [r * BEAMS for r in range(requests)]
    starts = np.concatenate([[0], np.cumsum([len(p) for p in prompts])]).tolist()
    x = search.forward([t for p in prompts for t in p], firsts, [i for p in prompts for i in range(len(p))], starts,
                       [len(p) for p in prompts], trace_of(firsts, starts))
    last = x[torch.tensor([s - 1 for s in starts[1:]], device=DEV)]
    # all beams start from the prompt: they share its logits, and only the first counts
    logits = search.logits(last).repeat_interleave(BEAMS, 0).contiguous()
    scores = torch.full((requests, BEAMS), -torch.inf, device=DEV)
    scores[:, 0] = 0
    lens = [len(p) for p in prompts for _ in range(BEAMS)]
    texts = [list(p) for p in prompts for _ in range(BEAMS)]

    for step in range(8):
        new, parents, tokens = (torch.empty(requests, BEAMS, dtype=t, device=DEV) for t in (torch.float32, torch.int32, torch.int32))
        ops.beam_select(engine, logits, scores, new, parents, tokens)
        want, at = _first(_reference(logits.cpu(), scores.cpu()), BEAMS)
        assert torch.equal(parents.cpu().long(), at // VOCAB) and torch.equal(tokens.cpu().long(), at % VOCAB), step
        assert torch.allclose(new.cpu().double(), want, rtol=1e-6, atol=1e-5)
        scores = new
        chosen = parents.view(-1).tolist()
        search.reorder(chosen, lens)
        source = [i // BEAMS * BEAMS + p for i, p in enumerate(chosen)]
        for h in (k_of, v_of):
            for layer in range(LAYERS):
                h[layer] = [h[layer][s] for s in source]
        texts = [texts[s] + [t] for s, t in zip(source, tokens.view(-1).tolist())]
        # every slot's rows are those of the beam that it went on from
        for layer in range(LAYERS):
            for slot in (0, 5, requests * BEAMS - 1):
                ko, vo = (torch.empty(lens[slot], KVH, HD, device=DEV) for _ in range(2))
                ops.kv_read_fp4(engine, *[c[layer] for c in search.caches], ko, vo, first_row=search.base[slot])
                assert torch.equal(ko.cpu().double(), k_of[layer][slot]) and torch.equal(vo.cpu().double(), v_of[layer][slot])
        # one decode step of all beams
        rows = requests * BEAMS
        x = search.forward([t[-1] for t in texts], list(range(rows)), lens, list(range(rows + 1)), [n + 1 for n in lens],
                           trace_of(range(rows), list(range(rows + 1))))
        lens = [n + 1 for n in lens]
        logits = search.logits(x)
    # beams of a request are different texts, best first
    for r in range(requests):
        mine = [tuple(t) for t in texts[r * BEAMS:(r + 1) * BEAMS]]
        assert len(set(mine)) == BEAMS
    assert (scores[:, :-1] >= scores[:, 1:]).all()
