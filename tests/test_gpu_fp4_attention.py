"""janus_fp4_attention against 64 bits, with the bounds of packed_ref (a 4-bit value is a binary16 number)."""
import math

import pytest
import torch

from janus_amd import ops
from fp4_ref import decode, random_cache
from packed_ref import attend, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f16": torch.float16, "f32": torch.float32}


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _case(heads, kvh, hd, seqs, dtype, cap=None, seed=0, sigma=1.5, behind=0, poison=True, lo=122, hi=129):
    """seqs: (rows, length) of each. Cache rows that no sequence owns hold NaN blocks."""
    gen = torch.Generator().manual_seed(seed)
    rows = sum(n for n, _ in seqs)
    cap = cap or max(1, max(m for _, m in seqs))
    q = (torch.randn(rows + behind, heads, hd, generator=gen) * sigma).to(dtype)
    cache = [*random_cache(gen, len(seqs) * cap + 1, kvh, hd, lo, hi), *random_cache(gen, len(seqs) * cap + 1, kvh, hd, lo, hi)]
    slots = torch.randperm(len(seqs), generator=gen).tolist()
    k, v = decode(*cache[:2]), decode(*cache[2:])
    if poison:
        for s, (_, m) in zip(slots, seqs):
            for c in cache[1::2]:
                c[s * cap + max(0, m):(s + 1) * cap] = 255
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    return q, [c.to(DEV) for c in cache], k, v, slots, starts, cap


def _run(engine, heads, kvh, hd, seqs, types, hint=0, scale=0.0, device="cpu", **kw):
    dtype = TYPES[types]
    q, cache, k, v, slots, starts, cap = _case(heads, kvh, hd, seqs, dtype, **kw)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=DEV)
    ops.fp4_attention(engine, q.to(DEV), *cache, out, len(seqs), cap, q_start=_i32(starts),
                      row_base=_i32([s * cap for s in slots]), seq_lens=_i32([m for _, m in seqs]), max_len_hint=hint,
                      scale=scale)
    engine.sync()
    for s, (n, m), i in zip(slots, seqs, starts):
        m = max(0, m)
        with torch.device(device):
            want, tol = attend(q[i:i + n].to(device), k[s * cap:s * cap + m].to(device), v[s * cap:s * cap + m].to(device),
                               [max(0, m - n + 1 + r) for r in range(n)], types == "f16", True, scale or None)
        check(out[i:i + n], want.cpu(), tol.cpu(), (types, heads, kvh, hd, n, m))
    assert (out[starts[-1]:] == 7.0).all()


LAYOUTS = [(4, 2, 64), (8, 2, 128), (3, 3, 128), (5, 1, 64), (8, 8, 128), (12, 4, 64)]


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
def test_one_row_of_each(engine, types, heads, kvh, hd):
    # a decode step: lengths at and around 16 and 32, none, one
    _run(engine, heads, kvh, hd, [(1, m) for m in (1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0, 130)], types)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
def test_whole_prompts(engine, types, heads, kvh, hd):
    _run(engine, heads, kvh, hd, [(1, 1), (31, 31), (0, 0), (32, 32), (33, 33), (2, 2), (129, 129), (200, 200)], types, behind=3)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (4, 4, 64), (12, 4, 128), (40, 8, 128), (16, 1, 128), (40, 1, 64)])
def test_rows_behind_a_context(engine, types, heads, kvh, hd):
    # chunks, drafted tokens and single tokens of one call
    _run(engine, heads, kvh, hd, [(5, 64), (1, 63), (1, 65), (64, 200), (7, 700), (40, 41), (1, 1)], types, behind=3)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_rows_that_see_nothing(engine, types):
    # fewer positions than rows: the first rows see none; lengths of zero and below
    _run(engine, 8, 2, 64, [(9, 4), (3, 0), (70, 2), (1, 0), (2, 2), (1, -5), (4, -1)], types, cap=80)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("heads,kvh,hd", [(32, 8, 128), (40, 1, 128), (32, 32, 128), (4, 2, 64), (16, 1, 128), (24, 8, 64)])
def test_long_context_is_split(engine, types, heads, kvh, hd):
    _run(engine, heads, kvh, hd, [(1, 2100)], types)
    _run(engine, heads, kvh, hd, [(1, 1900), (3, 333), (1, 5), (0, 0), (1, 0)], types, seed=1)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hint", [1, 100, 100000])
def test_hint_only_plans(engine, types, hint):
    _run(engine, 8, 2, 64, [(2, 1500), (130, 900)], types, hint=hint)
    _run(engine, 8, 8, 128, [(1, 1500), (1, 3)], types, hint=hint)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_many_sequences(engine, types):
    # more sequences than a wavefront has lanes, some without rows
    _run(engine, 4, 2, 64, [((i * 7) % 5, 3 + (i * 7) % 5 + i % 11) for i in range(150)], types, cap=24)
    _run(engine, 4, 4, 128, [(1, 1 + i * 13 % 90) for i in range(130)], types, cap=90)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("sigma", [0.0, 1e-6, 40.0])
def test_score_ranges(engine, types, sigma):
    # equal scores, tiny queries, and one position that takes nearly all weight
    _run(engine, 4, 2, 128, [(70, 300), (1, 200)], types, sigma=sigma)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_scales_of_many_binades(engine, types):
    _run(engine, 8, 2, 128, [(1, 300), (40, 90)], types, lo=114, hi=131, sigma=0.5, scale=0.01)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("size", [1e-30, 1e-3, 3e4])
def test_query_magnitudes(engine, types, size):
    """Rows of q from tiny to large, with a scale that makes their scores ordinary."""
    if types == "f16" and size < 1e-3:
        pytest.skip("not a binary16 number")
    _run(engine, 8, 2, 128, [(3, 120), (1, 700)], types, sigma=size / 3, scale=min(1e30, 0.3 / size))


def test_a_long_prompt(engine):
    _run(engine, 8, 2, 128, [(1500, 1500)], "f16", device=DEV)
    _run(engine, 8, 2, 128, [(700, 2000), (300, 300)], "f32", device=DEV)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_decode_step_without_tables(engine, types):
    """Without q_start every sequence has rows / nseq; without lengths as many positions as rows."""
    dtype = TYPES[types]
    gen = torch.Generator().manual_seed(11)
    heads, kvh, hd, cap = 8, 2, 64, 24
    q = torch.randn(12, heads, hd, generator=gen).to(dtype)
    cache = [*random_cache(gen, 4 * cap, kvh, hd), *random_cache(gen, 4 * cap, kvh, hd)]
    k, v = decode(*cache[:2]), decode(*cache[2:])
    dev = [c.to(DEV) for c in cache]
    out = torch.empty(12, heads, hd, dtype=dtype, device=DEV)
    ops.fp4_attention(engine, q.to(DEV), *dev, out, 4, cap)
    for s in range(4):
        want, tol = attend(q[3 * s:3 * s + 3], k[s * cap:s * cap + 3], v[s * cap:s * cap + 3], [1, 2, 3], types == "f16", True)
        check(out[3 * s:3 * s + 3], want, tol, s)
    out4 = torch.empty(4, heads, hd, dtype=dtype, device=DEV)
    ops.fp4_attention(engine, q[:4].to(DEV).contiguous(), *dev, out4, 4, cap, seq_lens=_i32([cap, 1, 7, 20]))
    for s, n in enumerate((cap, 1, 7, 20)):
        want, tol = attend(q[s:s + 1], k[s * cap:s * cap + n], v[s * cap:s * cap + n], [n], types == "f16", True)
        check(out4[s:s + 1], want, tol, s)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_lengths_beyond_the_slot_and_the_cache(engine, types):
    """Positions of max_seq_len and above, and cache rows beyond the cache, do not exist; nothing is read there."""
    dtype = TYPES[types]
    gen = torch.Generator().manual_seed(12)
    heads, kvh, hd = 4, 2, 64
    cache = [*random_cache(gen, 100, kvh, hd), *random_cache(gen, 100, kvh, hd)]
    k, v = decode(*cache[:2]), decode(*cache[2:])
    dev = [c.to(DEV) for c in cache]
    q = torch.randn(5, heads, hd, generator=gen).to(dtype)
    out = torch.empty(5, heads, hd, dtype=dtype, device=DEV)
    base, lens = [0, 90, 99, 200, -3], [50, 50, 2 ** 31 - 1, 10, 10]
    ops.fp4_attention(engine, q.to(DEV), *dev, out, 5, 40, row_base=_i32(base), seq_lens=_i32(lens))
    for s, n in enumerate((40, 10, 1, 0, 0)):
        want, tol = attend(q[s:s + 1], k[base[s]:base[s] + n] if n else k[:0], v[base[s]:base[s] + n] if n else v[:0], [n], types == "f16", True)
        check(out[s:s + 1], want, tol, s)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("rows,length", [(1, 40), (1, 2500), (6, 700), (90, 300)])
def test_nan_blocks(engine, types, rows, length):
    """A NaN block of K reaches every dim of the heads that read it, one of V its 32 dims;
    rows that do not see it are untouched. q with an infinity or NaN: NaN for its head."""
    heads, kvh, hd = 8, 4, 128
    q, cache, k, v, slots, starts, cap = _case(heads, kvh, hd, [(rows, length)], TYPES[types], seed=5)
    at = length - max(1, rows // 2)   # the last rows see it, with many rows the first do not
    cache[1][at, 0, 2] = 255
    cache[3][at, 2, 1] = 141
    cache[3][3, 3, 0] = 200
    q[rows - 1, 2, 7] = math.inf      # KV head 1
    out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
    ops.fp4_attention(engine, q.to(DEV), *cache, out, 1, cap, seq_lens=_i32([length]))
    got = out.float().cpu()
    clean = torch.where(torch.isfinite(q), q, 0)
    want, tol = attend(clean, k[:length], v[:length], [length - rows + 1 + r for r in range(rows)], types == "f16", True)
    sees = torch.tensor([length - rows + 1 + r > at for r in range(rows)])
    assert sees.any() and (rows == 1 or not sees.all())
    nan = torch.zeros(got.shape, dtype=torch.bool)
    nan[:, 0:2] = sees[:, None, None]
    nan[:, 4:6, 32:64] = sees[:, None, None]
    nan[:, 6:8, 0:32] = True
    nan[rows - 1, 2] = True
    assert torch.equal(got.isnan(), nan)
    got[nan] = want[nan].float()
    check(got, want, tol, (types, rows, length))


@pytest.mark.parametrize("types", sorted(TYPES))
def test_in_place_on_another_stream(engine, types):
    q, cache, k, v, slots, starts, cap = _case(8, 2, 64, [(1, 1300), (4, 90)], TYPES[types], seed=8)
    tables = dict(q_start=_i32(starts), row_base=_i32([s * cap for s in slots]), seq_lens=_i32([1300, 90]))
    want = torch.empty(q.shape, dtype=q.dtype, device=DEV)
    dev = q.to(DEV)
    ops.fp4_attention(engine, dev, *cache, want, 2, cap, **tables)
    engine.sync()
    stream = torch.cuda.Stream()
    engine.bind_stream(stream)
    try:
        ops.fp4_attention(engine, dev, *cache, dev, 2, cap, **tables)
        engine.sync()
    finally:
        engine.bind_stream(torch.cuda.default_stream())
    assert torch.equal(dev, want)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_captured_calls_follow_their_tables(engine, types):
    """A captured call, replayed with other lengths, equals the eager one; two graphs of one context share its workspace."""
    dtype = TYPES[types]
    heads, kvh, hd, cap = 8, 2, 128, 1500
    q, cache, k, v, slots, starts, _ = _case(heads, kvh, hd, [(1, cap), (1, cap), (1, cap)], dtype, seed=9)
    q2 = torch.randn(3 * 40, heads, hd, generator=torch.Generator().manual_seed(10)).to(dtype).to(DEV)
    dev, base, lens = q.to(DEV), _i32([s * cap for s in slots]), _i32([5, 700, cap])
    out, out2 = torch.zeros_like(dev), torch.zeros_like(q2)

    def step():
        ops.fp4_attention(engine, dev, *cache, out, 3, cap, row_base=base, seq_lens=lens)

    def chunk():
        ops.fp4_attention(engine, q2, *cache, out2, 3, cap, row_base=base, seq_lens=lens)

    stream = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(stream):
        engine.bind_stream(stream)
        try:
            for call in (step, chunk):
                call()
                stream.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=stream):
                    call()
                graphs.append(g)
            for new in ([5, 700, cap], [1, 1, 1], [cap, 0, 33], [40, 1200, 64]):
                lens.copy_(_i32(new))
                got = []
                for g, o in zip(graphs, (out, out2)):
                    o.fill_(3)
                    g.replay()
                for o in (out, out2):
                    got.append(o.clone())
                step()
                chunk()
                stream.synchronize()
                assert torch.equal(got[0], out) and torch.equal(got[1], out2), new
        finally:
            engine.bind_stream(torch.cuda.default_stream())


def test_runs_repeat(engine):
    """The same call twice gives the same bits."""
    for types, seqs in (("f16", [(1, 3000), (1, 40)]), ("f32", [(3, 900), (50, 60)])):
        q, cache, k, v, slots, starts, cap = _case(8, 8, 128, seqs, TYPES[types], seed=13)
        outs = []
        for _ in range(2):
            out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
            ops.fp4_attention(engine, q.to(DEV), *cache, out, len(seqs), cap, q_start=_i32(starts),
                              row_base=_i32([s * cap for s in slots]), seq_lens=_i32([m for _, m in seqs]))
            outs.append(out)
        assert torch.equal(*outs)


def test_offsets_beyond_32_bits(engine):
    """A slot whose values lie beyond 2^32 bytes."""
    heads, kvh, hd, n = 32, 32, 128, 70
    rows = 2 ** 32 // (kvh * hd // 2) + n
    gen = torch.Generator().manual_seed(14)
    part = [*random_cache(gen, n, kvh, hd), *random_cache(gen, n, kvh, hd)]
    cache = []
    for p in part:
        c = torch.zeros(rows, *p.shape[1:], dtype=torch.uint8, device=DEV)
        c[rows - n:] = p.to(DEV)
        cache.append(c)
    q = torch.randn(1, heads, hd, generator=gen)
    out = torch.empty(1, heads, hd, device=DEV)
    ops.fp4_attention(engine, q.to(DEV), *cache, out, 1, n, row_base=_i32([rows - n]), seq_lens=_i32([n]))
    want, tol = attend(q, decode(*part[:2]), decode(*part[2:]), [n], False, True)
    check(out, want, tol)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_rows_that_see_nothing_of_a_split_context(engine, types):
    _run(engine, 8, 2, 128, [(40, 1500), (40, 0), (40, 33)], types, cap=1500)
    _run(engine, 8, 8, 64, [(2, 1000), (2, 1), (1, 0), (9, 70)], types)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("rows", [3, 20, 70])
def test_scores_beyond_their_own_last_bits(engine, types, rows):
    """Scores whose spacing is far above 1: the farthest ahead takes all weight, equal ones share it."""
    dtype = TYPES[types]
    gen = torch.Generator().manual_seed(21)
    hd, n, size = 128, 1100, 3e4 if types == "f16" else 1e8
    q = (torch.randn(rows, 2, hd, generator=gen).sign() * size).to(dtype)
    cache = random_cache(gen, n, 1, hd, 127, 128), random_cache(gen, n, 1, hd)
    codes = torch.where(torch.rand(n, 1, hd // 2, generator=gen) < 0.5, 0x66, 0xEE) ^ torch.where(
        torch.rand(n, 1, hd // 2, generator=gen) < 0.5, 0x80, 0)   # 4 and -4
    k, v = decode(codes.to(torch.uint8), cache[0][1]), decode(*cache[1])
    k, v = k * 16, v   # scale byte 131
    dev = [c.to(DEV) for c in (codes.to(torch.uint8), cache[0][1] + 4, *cache[1])]
    out = torch.empty(q.shape, dtype=dtype, device=DEV)
    ops.fp4_attention(engine, q.to(DEV), *dev, out, 1, n, seq_lens=_i32([n]))
    s = torch.einsum("rhd,jd->rhj", q.double(), k[:, 0])
    for r in range(rows):
        seen = s[r, :, :n - rows + 1 + r]
        first = (seen == seen.amax(-1, keepdim=True)).double()
        want = first @ v[:seen.shape[1], 0] / first.sum(-1, keepdim=True)
        tol = 2.0 ** (-10 if types == "f16" else -20) * v.abs().max()
        check(out[r], want, tol.expand_as(want), (types, r))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("rows,n,at", [(1, 200, 69), (20, 200, 69), (20, 200, 104), (40, 200, 69), (1, 8192, 6000),
                                       (20, 6000, 4011), (40, 6000, 4011)])
def test_a_maximum_that_rises_by_its_last_bit(engine, types, rows, n, at):
    """Of two scores next to each other in 32 bits, near 2^31 before the scale, the later one is 16 powers of two
    ahead. Of m = 65504 2^15 + 128 x, with this x, scale log2(e) m rounded to a multiple of 32 hides more than 14.3 of
    them from an exponent that is taken as scale log2(e) s less that. In one step or the next, another phase, another share."""
    dtype, x, hd = TYPES[types], 40, 128
    q = torch.zeros(rows, 2, hd, dtype=dtype)
    q[..., 0], q[..., 32], q[..., 64] = 65504.0, x, 1.0
    codes, scales = torch.zeros(n, 1, hd // 2, dtype=torch.uint8), torch.full((n, 1, hd // 32), 132, dtype=torch.uint8)
    codes[[0, at], 0, 0], codes[[0, at], 0, 16], codes[at, 0, 32] = 6, 6, 6   # 4 times the block's scale
    scales[:, :, 0] = 140
    cache = random_cache(torch.Generator().manual_seed(22), n, 1, hd)
    k, v = decode(codes, scales)[:, 0], decode(*cache)[:, 0]
    s = k @ q[0, 0].double()
    assert s[0] == 65504 * 2.0 ** 15 + 128 * x and s[at] == s[0] + 128 and (s.float() == s).all()
    out = torch.empty(q.shape, dtype=dtype, device=DEV)
    ops.fp4_attention(engine, q.to(DEV), *[c.to(DEV) for c in (codes, scales, *cache)], out, 1, n, seq_lens=_i32([n]))
    w = math.exp(-128 / math.sqrt(hd))
    want = (v[at] + w * v[0]) / (1 + w)
    # the output's own rounding (w v[0] alone is below 2^-14, where binary16 has steps of 2^-24), and the weights': w is
    # below 2^-16, and its binary16 part off by 2^-11 of itself
    tol = want.abs() * torch.finfo(dtype).eps + (v[at].abs() + v[0].abs()) * 2.0 ** -22 + (2.0 ** -25 if types == "f16" else 0)
    check(out.flatten(0, 1), want.expand(2 * rows, hd), tol.expand(2 * rows, hd), (types, rows))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("heads,kvh,hd,n", [(16, 2, 64, 2), (17, 1, 128, 1), (32, 1, 64, 1), (32, 2, 128, 1), (33, 3, 64, 1),
                                            (40, 8, 128, 6), (12, 3, 128, 32), (4, 1, 64, 33), (10, 5, 128, 20)])
def test_columns_at_the_kernels_borders(engine, types, heads, kvh, hd, n):
    """16 and 17 columns of a sequence, 32 and 33, 128 and more, behind contexts that are split and that are not."""
    for context in (0, 77, 1400):
        _run(engine, heads, kvh, hd, [(n, context + n), (n, n), (max(1, n - 1), context // 2 + n)], types, seed=context)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("heads,kvh,n", [(8, 8, 1), (4, 1, 12), (4, 1, 20)])
def test_many_sequences_share_a_split_context(engine, types, heads, kvh, n):
    """More sequences than lanes on the split path; their slots overlap, as prompts with a common beginning may."""
    gen = torch.Generator().manual_seed(31)
    dtype, hd, nseq, cap = TYPES[types], 128, 130, 1500
    cache = [*random_cache(gen, 2 * cap, kvh, hd), *random_cache(gen, 2 * cap, kvh, hd)]
    k, v = decode(*cache[:2]), decode(*cache[2:])
    q = torch.randn(nseq * n, heads, hd, generator=gen).to(dtype)
    base = torch.randint(0, cap, (nseq,), generator=gen).tolist()
    lens = torch.randint(n, cap + 1, (nseq,), generator=gen).tolist()
    lens[3], lens[70], lens[129] = 0, cap, 1
    out = torch.empty(q.shape, dtype=dtype, device=DEV)
    ops.fp4_attention(engine, q.to(DEV), *[c.to(DEV) for c in cache], out, nseq, cap, row_base=_i32(base), seq_lens=_i32(lens))
    for s in (*range(0, nseq, 9), 3, 70, 129):
        b, m = base[s], lens[s]
        want, tol = attend(q[s * n:(s + 1) * n], k[b:b + m], v[b:b + m], [max(0, m - n + 1 + r) for r in range(n)], types == "f16", True)
        check(out[s * n:(s + 1) * n], want, tol, (types, s, m))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("rows", [12, 40])
def test_nan_blocks_of_a_split_context(engine, types, rows):
    """Many columns and shares: a NaN of K for the rows from it on, one of V in its dims, others as they were."""
    heads, kvh, hd, length = 8, 2, 128, 2600
    q, cache, k, v, slots, starts, cap = _case(heads, kvh, hd, [(rows, length)], TYPES[types], seed=6)
    at = length - 11
    cache[1][at, 0, 3] = 255
    cache[3][1700, 1, 2] = 141
    out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
    ops.fp4_attention(engine, q.to(DEV), *cache, out, 1, cap, seq_lens=_i32([length]))
    got = out.float().cpu()
    want, tol = attend(q, k[:length], v[:length], [length - rows + 1 + r for r in range(rows)], types == "f16", True)
    nan = torch.zeros(got.shape, dtype=torch.bool)
    nan[rows - 11:, 0:4] = True
    nan[:, 4:8, 64:96] = True
    assert torch.equal(got.isnan(), nan)
    got[nan] = want[nan].float()
    check(got, want, tol, types)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_two_contexts_at_once(engine, types):
    """Split calls of two contexts on two streams, side by side: each has its own workspace."""
    other = ops.ComputeEngine(0)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    cases = [_case(8, 2, 128, [(1, 3000), (1, 70)], TYPES[types], seed=41), _case(8, 8, 128, [(6, 2500)], TYPES[types], seed=42)]
    lens = [_i32([3000, 70]), _i32([2500])]
    try:
        q = [c[0].to(DEV) for c in cases]
        base = [_i32([s * c[6] for s in c[4]]) for c in cases]
        want = [torch.empty_like(x) for x in q]
        for i in range(2):
            ops.fp4_attention(engine, q[i], *cases[i][1], want[i], len(lens[i]), cases[i][6], row_base=base[i], seq_lens=lens[i])
        outs = [[torch.empty_like(x) for _ in range(8)] for x in q]
        torch.cuda.synchronize()
        engine.bind_stream(streams[0])
        other.bind_stream(streams[1])
        for t in range(8):
            for i, e in enumerate((engine, other)):
                ops.fp4_attention(e, q[i], *cases[i][1], outs[i][t], len(lens[i]), cases[i][6], row_base=base[i], seq_lens=lens[i])
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(o, want[i]) for o in outs[i])
    finally:
        engine.bind_stream(torch.cuda.default_stream())
        other.close()


def test_rows_of_wider_tensors(engine):
    """Rows of larger tensors: what lies beside them stays."""
    heads, kvh, hd = 4, 2, 64
    q, cache, k, v, slots, starts, cap = _case(heads, kvh, hd, [(3, 90)], torch.float16, seed=17)
    wide = torch.full((5, heads, hd), 9.0, dtype=torch.float16, device=DEV)
    wide[1:4] = q.to(DEV)
    out = torch.full((5, heads, hd), 3.0, dtype=torch.float16, device=DEV)
    ops.fp4_attention(engine, wide[1:4], *cache, out[1:4], 1, cap, seq_lens=_i32([90]))
    want, tol = attend(q, k[:90], v[:90], [88, 89, 90], True, True)
    check(out[1:4], want, tol)
    assert (out[[0, 4]] == 3).all()


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("rows,at", [(1, 3), (1, 4990), (20, 3)])
@pytest.mark.parametrize("hd", [64, 128])
def test_weights_that_are_small_in_binary16(engine, types, rows, at, hd):
    """One position 2^22 ahead of 4999 equal ones, whose weights are subnormal in binary16: together they count, in
    the sum as in the output. A weight is off by half of 2^-24 / 2^-15 at most, the output by that and its own rounding."""
    dtype, n = TYPES[types], 5000
    q = torch.zeros(rows, 1, hd, dtype=dtype)
    q[:, 0, 0] = 22 * math.log(2)
    kc, vc = torch.zeros(n, 1, hd // 2, dtype=torch.uint8), torch.full((n, 1, hd // 2), 0x22, dtype=torch.uint8)
    kc[at, 0, 0], vc[at] = 0x02, 0
    one = torch.full((n, 1, hd // 32), 127, dtype=torch.uint8)
    for values, tol in ((vc, 2.0 ** -9), (vc ^ 0x22, 2.0 ** -11)):   # of the many, of the one: w / (1 + w) and 1 / (1 + w)
        out = torch.empty(rows, 1, hd, dtype=dtype, device=DEV)
        ops.fp4_attention(engine, q.to(DEV), *(x.to(DEV) for x in (kc, one, values, one)), out, 1, n, seq_lens=_i32([n]), scale=1.0)
        for r in range(rows):
            w = (n - rows + r) * math.exp(-float(q[r, 0, 0]))
            want = (w if values is vc else 1.0) / (1 + w)
            assert (out[r].double().cpu() / want - 1).abs().max() < tol, (r, out[r].flatten()[:4], want)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("sigma", [1.5, 40.0])
def test_more_tiles_than_cus(engine, types, hd, sigma):
    # 384 tiles of 128 columns and more: prompts of odd lengths, chunks behind a context, one row, none, more rows than positions
    seqs = [(70, 70), (129, 129), (65, 200), (1, 300), (0, 0), (90, 65), (64, 64), (127, 127)]
    _run(engine, 64, 32, hd, seqs, types, behind=2, sigma=sigma, device=DEV)


@pytest.mark.parametrize("rows", [40, 70])
def test_many_tiles_in_parts(engine, rows):
    # 32 tiles of each of eight heads, 80 or 140 columns: binary16 rows behind a long context
    _run(engine, 16, 8, 128, [(rows, 1900 + 30 * i) for i in range(16)], "f16", device=DEV)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_nan_blocks_of_many_tiles(engine, types):
    heads, kvh, hd, n = 64, 32, 128, 150
    dtype = TYPES[types]
    gen = torch.Generator().manual_seed(31)
    q = torch.randn(5 * n, heads, hd, generator=gen).to(dtype)
    cache = [*random_cache(gen, 5 * n, kvh, hd), *random_cache(gen, 5 * n, kvh, hd)]
    cache[1][n + 100, 3, 1] = 255       # K of sequence 1, head 3
    cache[3][2 * n + 37, 5, 2] = 255    # V of sequence 2, head 5
    k, v = decode(*cache[:2]), decode(*cache[2:])
    out = torch.empty(q.shape, dtype=dtype, device=DEV)
    ops.fp4_attention(engine, q.to(DEV), *[c.to(DEV) for c in cache], out, 5, n)
    odd = torch.zeros(5 * n, heads, hd, dtype=torch.bool)
    odd[n + 100:2 * n, 6:8] = True
    odd[2 * n + 37:3 * n, 10:12, 64:96] = True
    got = out.cpu()
    assert torch.equal(got.isnan(), odd)
    for s in (0, 1, 2, 4):
        at = slice(s * n, (s + 1) * n)
        with torch.device(DEV):
            want, tol = attend(q[at].to(DEV), k[at].nan_to_num(0).to(DEV), v[at].nan_to_num(0).to(DEV),
                               list(range(1, n + 1)), types == "f16", True, None)
        fine = ~odd[at]
        check(got[at][fine], want.cpu()[fine], tol.cpu()[fine], (types, s))


@pytest.mark.parametrize("types", sorted(TYPES))
def test_far_scores_of_many_tiles(engine, types):
    """As test_scores_beyond_their_own_last_bits, 32 KV heads of 140 columns, 4 sequences."""
    dtype = TYPES[types]
    gen = torch.Generator().manual_seed(33)
    hd, kvh, n, size = 128, 32, 70, 3e4 if types == "f16" else 1e8
    q = (torch.randn(4 * n, 2 * kvh, hd, generator=gen).sign() * size).to(dtype)
    codes = torch.where(torch.rand(4 * n, kvh, hd // 2, generator=gen) < 0.5, 0x66, 0xEE).to(torch.uint8)   # 4 and -4
    scales = torch.full((4 * n, kvh, hd // 32), 131, dtype=torch.uint8)
    values = random_cache(gen, 4 * n, kvh, hd)
    k, v = decode(codes, scales), decode(*values)
    out = torch.empty(q.shape, dtype=dtype, device=DEV)
    ops.fp4_attention(engine, q.to(DEV), *[c.to(DEV) for c in (codes, scales, *values)], out, 4, n)
    got = out.cpu()
    for s in (0, 3):
        for h in (0, 7, 63):
            at = slice(s * n, (s + 1) * n)
            score = q[at, h].double() @ k[at, h // 2].t()
            score = score.masked_fill(torch.ones(n, n).triu(1).bool(), -math.inf)
            first = (score == score.amax(-1, keepdim=True)).double()
            want = first @ v[at, h // 2] / first.sum(-1, keepdim=True)
            tol = 2.0 ** (-10 if types == "f16" else -20) * v.abs().max()
            check(got[at, h], want, tol.expand_as(want), (types, s, h))
