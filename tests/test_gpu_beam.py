"""janus_beam_select against 64 bits, janus_kv_reorder against a copy."""
import math

import pytest
import torch

from janus_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _reference(logits, scores):
    """Values [batch, beams * vocab] in 64 bits, by the operator's rules."""
    batch, beams = scores.shape
    x = logits.double().view(batch, beams, -1)
    s = scores.double()[..., None]
    lse = torch.logsumexp(x, -1, keepdim=True)
    value = s + (x - lse)
    odd = x.isnan().any(-1, keepdim=True) | (x == math.inf).any(-1, keepdim=True) | s.isnan() | (s == math.inf)
    value = torch.where(odd, math.nan, value)
    ended = (s == -math.inf) | ((x == -math.inf).all(-1, keepdim=True) & ~odd)
    return torch.where(ended, -math.inf, value).view(batch, -1)


def _first(value, n):
    """The n largest, NaN above all, equal ones by index: (values, indices)."""
    key = torch.where(value.isnan(), math.inf, value)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :n]
    return value.gather(1, order), order


def _select(engine, logits, scores, n):
    batch = scores.shape[0]
    out = torch.empty(batch, n, device=DEV)
    parents, tokens = (torch.full((batch, n), -7, dtype=torch.int32, device=DEV) for _ in range(2))
    ops.beam_select(engine, logits.to(DEV), scores.to(DEV), out, parents, tokens)
    return out.cpu(), parents.cpu(), tokens.cpu()


def _check(engine, logits, scores, n):
    vocab = logits.shape[-1]
    out, parents, tokens = _select(engine, logits, scores, n)
    want, at = _first(_reference(logits, scores), n)
    assert torch.equal(parents.long(), at // vocab) and torch.equal(tokens.long(), at % vocab)
    # each term of the sum: the difference to the maximum is rounded (|t| u of the term, at most log V u of the
    # sum), its exponential off by a few u; 32 terms are added in binary32; the value is rounded once
    tol = (48 + math.log(vocab)) * U + want.abs() * U
    off = (out.double() - want).abs()
    fine = torch.isfinite(want)
    assert (off[fine] <= tol[fine]).all(), float((off / tol)[fine].max())
    assert torch.equal(out[~fine].double().nan_to_num(5), want[~fine].nan_to_num(5))


@pytest.mark.parametrize("batch,beams,vocab,n", [(1, 1, 1, 1), (1, 4, 128256, 8), (3, 5, 8193, 10), (2, 16, 8192, 64),
                                                 (7, 2, 1001, 3), (2, 64, 50, 64), (1, 3, 7, 21), (4, 8, 32000, 16),
                                                 (2, 1, 20000, 64), (1, 2, 300000, 64), (33, 3, 515, 6)])
@pytest.mark.parametrize("sigma", [0.5, 6.0])
def test_random_logits(engine, batch, beams, vocab, n, sigma):
    gen = torch.Generator().manual_seed(vocab + n)
    logits = torch.randn(batch * beams, vocab, generator=gen) * sigma
    scores = -5 * torch.rand(batch, beams, generator=gen)
    _check(engine, logits, scores, n)


@pytest.mark.parametrize("vocab", [60, 4000, 30001])
@pytest.mark.parametrize("n", [1, 12, 64])
def test_ties_go_to_the_lowest_index(engine, vocab, n):
    """Logits of few values, equal beams, constant logits: masses of equal values."""
    gen = torch.Generator().manual_seed(vocab)
    n = min(n, 3 * vocab)
    levels = torch.randint(0, 3, (3, vocab), generator=gen).float()
    _check(engine, levels, torch.tensor([[-1.0, -1.5, -1.0]]), n)
    _check(engine, levels[:1].expand(3, -1).contiguous(), torch.full((1, 3), -2.0), n)
    for value in (0.0, -0.0, 5.0, -1e30):
        _check(engine, torch.full((3, vocab), value), torch.tensor([[-1.0, 0.0, -1.0]]), n)
    mixed = torch.where(torch.rand(3, vocab, generator=gen) < 0.5, 0.0, -0.0)
    _check(engine, mixed, torch.zeros(1, 3), n)


@pytest.mark.parametrize("beams,vocab", [(16, 40000), (64, 50001)])
def test_many_parts_of_many_candidates(engine, beams, vocab):
    """64 candidates of each of 80 and 448 parts: the best of all in one part, in one beam, everywhere alike."""
    gen = torch.Generator().manual_seed(beams)
    logits = torch.randn(2 * beams, vocab, generator=gen)
    scores = -2 * torch.rand(2, beams, generator=gen)
    _check(engine, logits, scores, 64)
    one = logits.clone()
    one[3, 8192:8300] += 30       # 64 of one part before all others of its beam
    one[beams + 5, 7:20000:190] += 30
    _check(engine, one, scores, 64)
    _check(engine, logits, torch.where(torch.arange(beams) == 7, 0.0, scores - 40.0), 64)
    levels = torch.randint(0, 2, (2 * beams, vocab), generator=gen).float()
    _check(engine, levels, torch.full((2, beams), -1.0), 64)
    ended = scores.clone()
    ended[0, 1:] = ended[1] = -math.inf
    _check(engine, logits, ended, 64)
    logits[9, 3] = math.nan
    _check(engine, logits, scores, 64)


@pytest.mark.parametrize("order", [1, -1])
def test_sorted_logits(engine, order):
    # the best ones lie in few lanes and in one wavefront
    logits = torch.linspace(-9 * order, 9 * order, 20000)
    _check(engine, torch.stack([logits, logits.roll(777)]), torch.tensor([[0.0, -0.25]]), 64)
    every = torch.zeros(2, 16384)
    every[:, 5::256] = torch.arange(64.0) + 10   # one lane of each wavefront has all the best
    every[:, 6::256] = 100 - torch.arange(64.0)
    _check(engine, every, torch.tensor([[0.0, -0.5]]), 64)


def test_ended_beams(engine):
    """The first step (all beams but one have not begun), beams that have ended, all of them; their logits are not looked at."""
    gen = torch.Generator().manual_seed(2)
    logits = torch.randn(8, 9000, generator=gen)
    inf = math.inf
    for scores in ([[0, -inf, -inf, -inf], [-inf, -1, -inf, -2]], [[-inf] * 4, [-inf, -inf, -inf, -0.5]]):
        _check(engine, logits, torch.tensor(scores), 8)
    logits[1] = math.nan
    logits[2] = inf
    out, parents, tokens = _select(engine, logits, torch.tensor([[0, -inf, -inf, -1], [-1.0, -1, -1, -1]]), 8)
    assert torch.isfinite(out).all() and not ((parents[0] == 1) | (parents[0] == 2)).any()


def test_masked_tokens(engine):
    """-infinity among the logits: fewer tokens than asked for, one, none."""
    logits = torch.full((4, 9000), -math.inf)
    logits[0, [5, 8999]] = torch.tensor([1.0, 2.0])
    logits[1, 4000] = -3.0
    logits[3, 10:13] = 0.5
    _check(engine, logits, torch.tensor([[-1.0, -2.0, -1.0, -8.0]]), 16)
    _check(engine, logits, torch.tensor([[-1.0, -2.0], [-1.0, -8.0]]), 5)
    _check(engine, torch.full((2, 100), -math.inf), torch.zeros(1, 2), 64)


def test_values_that_are_not_finite(engine):
    """A beam with a NaN or +infinity among its logits or as its score has NaN for every token, and comes first."""
    gen = torch.Generator().manual_seed(3)
    for bad in (math.nan, math.inf):
        for at in (0, 4097, 8999):
            logits = torch.randn(3, 9000, generator=gen)
            logits[1, at] = bad
            _check(engine, logits, torch.tensor([[0.0, -50.0, -1.0]]), 6)
        _check(engine, torch.randn(3, 9000, generator=gen), torch.tensor([[0.0, -50.0, bad]]), 6)
    logits = torch.randn(2, 40, generator=gen)
    logits[0] = math.nan
    _check(engine, logits, torch.zeros(1, 2), 60)


def test_extreme_logits(engine):
    logits = torch.randn(2, 5000, generator=torch.Generator().manual_seed(4))
    logits[0] *= 1e30
    logits[1] = -3e38
    logits[1, 7] = -2.9e38
    _check(engine, logits, torch.tensor([[-1.0, -1.5]]), 12)
    _check(engine, logits * 1e-38, torch.tensor([[-1e30, 2e30]]), 12)


def test_selection_captured(engine):
    gen = torch.Generator().manual_seed(5)
    logits, scores = torch.randn(8, 20000, generator=gen).to(DEV), -torch.rand(2, 4, generator=gen).to(DEV)
    out, parents, tokens = (torch.empty(2, 8, dtype=t, device=DEV) for t in (torch.float32, torch.int32, torch.int32))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        engine.bind_stream(stream)
        try:
            ops.beam_select(engine, logits, scores, out, parents, tokens)
            stream.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                ops.beam_select(engine, logits, scores, out, parents, tokens)
            for i in range(4):
                logits.copy_(torch.randn(8, 20000, generator=gen).to(DEV))
                out.zero_()
                g.replay()
                stream.synchronize()
                want, at = _first(_reference(logits.cpu(), scores.cpu()), 8)
                assert torch.equal(tokens.cpu().long(), at % 20000) and torch.equal(parents.cpu().long(), at // 20000), i
        finally:
            engine.bind_stream(torch.cuda.default_stream())


# ---- reordering -------------------------------------------------------------------

def _reorder(engine, caches, beams, max_seq, base, parents, lens, layers):
    want = [c.clone() for c in caches]
    rows = caches[0].shape[1 if layers else 0]
    for i, p in enumerate(parents):
        if not 0 <= p < beams:
            continue
        src, dst = base[i // beams * beams + p], base[i]
        n = min(max_seq if lens is None else lens[i], max_seq, rows - max(src, dst))
        if src < 0 or dst < 0 or n <= 0:
            continue
        for c, w in zip(caches, want):
            if layers:
                w[:, dst:dst + n] = c[:, src:src + n]
            else:
                w[dst:dst + n] = c[src:src + n]
    dev = [c.to(DEV) for c in caches]
    ops.kv_reorder(engine, dev, beams, max_seq, _i32(base), _i32(parents), seq_lens=None if lens is None else _i32(lens),
                   layers=layers)
    for got, w in zip(dev, want):
        assert torch.equal(got.cpu(), w)


def _random(gen, shape, dtype):
    return torch.randint(0, 256, (*shape[:-1], shape[-1] * torch.empty(0, dtype=dtype).element_size()), generator=gen,
                         dtype=torch.uint8).view(dtype) if dtype != torch.float16 and dtype != torch.float32 \
        else torch.randn(shape, generator=gen).to(dtype)


@pytest.mark.parametrize("beams", [2, 3, 4, 7, 8, 13, 16, 17, 32])
@pytest.mark.parametrize("kind", ["f16", "f32", "fp4", "odd"])
def test_reorder(engine, beams, kind):
    gen = torch.Generator().manual_seed(beams)
    cap, groups, layers = 37, 3, 2
    rows = groups * beams * cap
    shapes = {"f16": [((2, 64), torch.float16)] * 2, "f32": [((3, 32), torch.float32)] * 2,
              "fp4": [((2, 32), torch.uint8), ((2, 2), torch.uint8)] * 2, "odd": [((1, 17), torch.uint8), ((5, 1), torch.int16)]}[kind]
    caches = [_random(gen, (layers, rows, *s), t) for s, t in shapes]
    slots = torch.randperm(groups * beams, generator=gen).tolist()
    base = [s * cap for s in slots]
    parents = torch.randint(0, beams, (groups * beams,), generator=gen).tolist()
    lens = torch.randint(0, cap + 1, (groups * beams,), generator=gen).tolist()
    _reorder(engine, caches, beams, cap, base, parents, lens, layers)
    _reorder(engine, [c[1].contiguous() for c in caches], beams, cap, base, parents, None, 0)


def test_permutations_and_forks(engine):
    gen = torch.Generator().manual_seed(1)
    cap, beams = 900, 6
    caches = [torch.randn(3, beams * cap, 4, 64, generator=gen).half() for _ in range(2)]
    base = [i * cap for i in range(beams)]
    for parents in ([1, 2, 3, 4, 5, 0], [5, 4, 3, 2, 1, 0], [0] * 6, [3] * 6, list(range(6)), [1, 0, 2, 2, 5, 4]):
        _reorder(engine, caches, beams, cap, base, parents, [cap, 1, 0, 513, 899, 64], 3)


def test_slots_that_stay(engine):
    """Parents outside the request, padding, empty slots, and slots that end with the cache."""
    gen = torch.Generator().manual_seed(2)
    caches = [torch.randn(65, 2, 32, generator=gen) for _ in range(2)]
    base, parents, lens = [0, 10, 20, -1, 30, 60, 40, 50], [1, -1, 4, 0, 3, 0, 1, 2 ** 31 - 1], [5, 9, 9, 9, 9, 10, 10, 5]
    _reorder(engine, caches, 4, 10, base, parents, lens, 0)
    _reorder(engine, caches, 8, 10, [0, 10, 20, 30, 60, -10, 40, -2 ** 31], [4, 5, 8, 0, 3, 0, 1, 2], [9] * 8, 0)


def test_reorder_beyond_32_bits_and_captured(engine):
    """Slots whose bytes lie beyond 2^32 of their buffer; a captured call follows its tables."""
    cap, width = 64, 1 << 16
    rows = (1 << 32) // width + 4 * cap
    cache = torch.zeros(rows, width, dtype=torch.uint8, device=DEV)
    small = torch.arange(rows * 4, dtype=torch.int32, device=DEV).view(rows, 4)
    base = [rows - cap, rows - 2 * cap, rows - 3 * cap, 0]
    for i, b in enumerate(base):
        cache[b:b + cap] = i + 1
    tables = [_i32(base), _i32([1, 2, 0, 0]), _i32([cap, cap, cap, 10])]
    stream = torch.cuda.Stream()
    state = [1, 2, 3, 4]
    with torch.cuda.stream(stream):
        engine.bind_stream(stream)
        try:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                ops.kv_reorder(engine, [cache, small], 4, cap, tables[0], tables[1], seq_lens=tables[2])
            for parents in ([1, 2, 0, 3], [0, 0, 1, 3], [2, 1, 0, 3], [3, 1, 2, 3]):
                tables[1].copy_(_i32(parents))
                tables[2].fill_(cap)
                g.replay()
                stream.synchronize()
                state = [state[p] for p in parents]
                for b, v in zip(base, state):
                    assert (cache[b:b + cap] == v).all(), parents
        finally:
            engine.bind_stream(torch.cuda.default_stream())
    assert not cache[cap:cap + 100].any()
