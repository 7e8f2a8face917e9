"""janus_prompt_attention and janus_prefix_attention against 64 bits."""
import math

import pytest
import torch

from janus_amd import ops
from packed_ref import attend, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f16": (torch.float16, torch.float16), "f32_f16": (torch.float32, torch.float16),
         "f32": (torch.float32, torch.float32)}


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _rand(gen, *shape, dtype=torch.float32, sigma=1.0):
    return (torch.randn(*shape, generator=gen) * sigma).to(dtype)


def _prompt(engine, types, heads, kvh, hd, seqs, cap=None, seed=0, sigma=1.5, poison=True, behind=0, scale=0.0, hint=0,
            device="cpu"):
    """seqs: (rows, length) of each; cache rows that no sequence owns hold NaN and
    infinities. Checks every row and that the rows behind stay as they were."""
    qt, kt = TYPES[types]
    gen = torch.Generator().manual_seed(seed)
    rows = sum(n for n, _ in seqs)
    cap = cap or max(1, max(m for _, m in seqs))
    q = _rand(gen, rows + behind, heads, hd, dtype=qt, sigma=sigma)
    k = _rand(gen, len(seqs) * cap, kvh, hd, dtype=kt)
    v = _rand(gen, len(seqs) * cap, kvh, hd, dtype=kt)
    slots = torch.randperm(len(seqs), generator=gen).tolist()
    kc, vc = k.clone(), v.clone()
    if poison:
        for s, (_, m) in zip(slots, seqs):
            kc[s * cap + m:(s + 1) * cap] = math.nan
            vc[s * cap + m:(s + 1) * cap] = math.inf
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    out = torch.full(q.shape, 7.0, dtype=qt, device=DEV)
    ops.prompt_attention(engine, q.to(DEV), kc.to(DEV), vc.to(DEV), out, len(seqs), cap, q_start=_i32(starts),
                         row_base=_i32([s * cap for s in slots]), seq_lens=_i32([m for _, m in seqs]),
                         max_len_hint=hint, scale=scale)
    engine.sync()
    with torch.device(device):
        for s, (n, m), i in zip(slots, seqs, starts):
            want, tol = attend(q[i:i + n].to(device), k[s * cap:s * cap + m].to(device), v[s * cap:s * cap + m].to(device),
                               [max(0, m - n + 1 + r) for r in range(n)], qt == torch.float16, kt == torch.float16,
                               scale or None)
            check(out[i:i + n], want.cpu(), tol.cpu(), (types, n, m))
    assert (out[rows:] == 7.0).all()


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("heads,kvh,hd", [(4, 2, 64), (8, 2, 128), (3, 3, 128), (5, 1, 64)])
def test_whole_prompts(engine, types, heads, kvh, hd):
    _prompt(engine, types, heads, kvh, hd, [(1, 1), (31, 31), (0, 0), (32, 32), (33, 33), (2, 2), (129, 129)])


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (4, 4, 64), (12, 4, 128)])
def test_rows_behind_a_context(engine, types, heads, kvh, hd):
    # chunks, drafted tokens and single tokens of one call, lengths at and around tile ends
    _prompt(engine, types, heads, kvh, hd, [(5, 64), (1, 63), (1, 65), (64, 200), (7, 700), (40, 41), (1, 1)], behind=3)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_rows_that_see_nothing(engine, types):
    # fewer positions than rows: the first rows see none; a length of zero
    _prompt(engine, types, 8, 2, 64, [(9, 4), (3, 0), (70, 2), (1, 0), (2, 2)], cap=80)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("heads,kvh", [(32, 8), (40, 1), (200, 1)])
def test_long_context_is_split(engine, types, heads, kvh):
    # one row, and a few, against positions that several workgroups share; more heads than a tile has columns
    _prompt(engine, types, heads, kvh, 128, [(1, 2100), (3, 333)])


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hint", [1, 100, 100000])
def test_hint_only_plans(engine, types, hint):
    _prompt(engine, types, 8, 2, 64, [(2, 1500), (130, 900)], hint=hint)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_many_sequences(engine, types):
    # more sequences than a wavefront has lanes, some without rows
    _prompt(engine, types, 4, 2, 64, [((i * 7) % 5, 3 + (i * 7) % 5 + i % 11) for i in range(150)], cap=24)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("sigma", [0.0, 1e-6, 40.0])
def test_score_ranges(engine, types, sigma):
    # equal scores, tiny queries, and one position that takes nearly all weight
    _prompt(engine, types, 4, 2, 128, [(70, 300)], sigma=sigma)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("rows", [3, 70])
def test_scores_beyond_their_own_last_bits(engine, types, rows):
    """Scores whose spacing is far above 1: the farthest ahead takes all weight."""
    qt, kt = TYPES[types]
    gen = torch.Generator().manual_seed(21)
    hd, n, size = 128, 1100, 3e4 if qt == torch.float16 else 1e8
    q = (_rand(gen, rows, 2, hd).sign() * size).to(qt)
    k = _rand(gen, n, 1, hd).sign().to(kt) * 64
    v = _rand(gen, n, 1, hd, dtype=kt)
    out = torch.empty(q.shape, dtype=qt, device=DEV)
    ops.prompt_attention(engine, q.to(DEV), k.to(DEV), v.to(DEV), out, 1, n, seq_lens=_i32([n]))
    s = torch.einsum("rhd,jd->rhj", q.double(), k[:, 0].double())
    for r in range(rows):
        seen = s[r, :, :n - rows + 1 + r]
        top = seen.amax(-1, keepdim=True)
        first = (seen == top).double()   # equal ones share the weight
        want = first @ v[:seen.shape[1], 0].double() / first.sum(-1, keepdim=True)
        tol = 2.0 ** (-10 if qt == torch.float16 else -20) * v.abs().max().double()
        check(out[r], want, tol.expand_as(want), (types, r))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("rows", [2, 40])
def test_infinity_in_one_part_of_a_split_context(engine, types, rows):
    qt, kt = TYPES[types]
    gen = torch.Generator().manual_seed(22)
    heads, kvh, hd, n = 32, 8, 128, 3000
    q = _rand(gen, rows, heads, hd, dtype=qt)
    k, v = (_rand(gen, n, kvh, hd, dtype=kt) for _ in range(2))
    want, tol = attend(q, k, v, [n - rows + 1 + r for r in range(rows)], qt == torch.float16, kt == torch.float16)
    v[1500, 0, 5], v[200, 7, 9] = math.inf, math.nan
    out = torch.empty(q.shape, dtype=qt, device=DEV)
    ops.prompt_attention(engine, q.to(DEV), k.to(DEV), v.to(DEV), out, 1, n, seq_lens=_i32([n]))
    got = out.float().cpu()
    assert (got[:, :4, 5] == math.inf).all() and got[:, 28:, 9].isnan().all()
    got[:, :4, 5] = want[:, :4, 5].float()
    got[:, 28:, 9] = want[:, 28:, 9].float()
    check(got, want, tol + 2.0 ** -20 * want.abs(), types)


def test_rising_scores(engine):
    # the maximum moves with every tile: each rescales what came before
    for types, (qt, kt) in sorted(TYPES.items()):
        n, hd = 512, 64
        q = torch.ones(1, 1, hd, dtype=qt)
        k = (torch.arange(n)[:, None, None] / 16.0).expand(n, 1, hd).to(kt).contiguous()
        v = _rand(torch.Generator().manual_seed(1), n, 1, hd, dtype=kt)
        out = torch.empty(1, 1, hd, dtype=qt, device=DEV)
        ops.prompt_attention(engine, q.to(DEV), k.to(DEV), v.to(DEV), out, 1, n, seq_lens=_i32([n]), scale=0.05)
        want, tol = attend(q, k, v, [n], qt == torch.float16, kt == torch.float16, 0.05)
        check(out, want, tol, types)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_defaults(engine, types):
    # no tables: sequences of equal rows, whole prompts, slots of max_seq_len rows
    qt, kt = TYPES[types]
    gen = torch.Generator().manual_seed(3)
    nseq, n, cap, heads, kvh, hd = 3, 37, 50, 4, 2, 64
    q = _rand(gen, nseq * n, heads, hd, dtype=qt)
    k, v = (_rand(gen, nseq * cap, kvh, hd, dtype=kt) for _ in range(2))
    out = torch.empty(q.shape, dtype=qt, device=DEV)
    ops.prompt_attention(engine, q.to(DEV), k.to(DEV), v.to(DEV), out, nseq, cap)
    for s in range(nseq):
        want, tol = attend(q[s * n:(s + 1) * n], k[s * cap:s * cap + n], v[s * cap:s * cap + n], range(1, n + 1),
                           qt == torch.float16, kt == torch.float16)
        check(out[s * n:(s + 1) * n], want, tol, s)
    # K and V packed like q: the starts are the row bases
    starts = _i32([0, 20, 20, 111])
    ops.prompt_attention(engine, q.to(DEV), k[:111].to(DEV), v[:111].to(DEV), out, 3, 111, q_start=starts, row_base=starts)
    for i, j in ((0, 20), (20, 111)):
        want, tol = attend(q[i:j], k[i:j], v[i:j], range(1, j - i + 1), qt == torch.float16, kt == torch.float16)
        check(out[i:j], want, tol, i)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_masked_infinities_stay_out(engine, types):
    """Infinities and NaN of K and V at positions that some rows see: the rows
    before them keep their values, the rows behind get the infinity or NaN of V in
    its dim alone, and a NaN of K everywhere."""
    qt, kt = TYPES[types]
    gen = torch.Generator().manual_seed(5)
    n, heads, kvh, hd = 100, 4, 2, 128
    q = _rand(gen, n, heads, hd, dtype=qt)
    k, v = (_rand(gen, n, kvh, hd, dtype=kt) for _ in range(2))
    clean, tol = attend(q, k, v, range(1, n + 1), qt == torch.float16, kt == torch.float16)
    v[70, 0, 5], v[71, 0, 6], v[72, 1, 7] = math.inf, -math.inf, math.nan
    k[90, 1, 0] = math.nan
    out = torch.empty(q.shape, dtype=qt, device=DEV)
    ops.prompt_attention(engine, q.to(DEV), k.to(DEV), v.to(DEV), out, 1, n)
    got = out.float().cpu()
    ok = torch.ones(n, heads, hd, dtype=torch.bool)
    ok[70:, :2, 5] = ok[71:, :2, 6] = ok[72:, 2:, 7] = False
    ok[90:, 2:] = False
    check(torch.where(ok, got.double(), 0.0), torch.where(ok, clean, 0.0), tol, types)
    assert (got[70:, :2, 5] == math.inf).all() and (got[71:, :2, 6] == -math.inf).all()
    assert got[72:, 2:, 7].isnan().all() and got[90:, 2:].isnan().all()


def test_infinite_keys(engine):
    """A key of -infinity (in the direction of q) has no weight; NaN rows of q
    stay in their rows."""
    for types, (qt, kt) in sorted(TYPES.items()):
        gen = torch.Generator().manual_seed(6)
        n, hd = 40, 64
        q = _rand(gen, n, 2, hd, dtype=qt).abs() + 0.5
        k, v = (_rand(gen, n, 1, hd, dtype=kt) for _ in range(2))
        k[3, 0, 9] = -math.inf
        q[17, 1] = math.nan
        out = torch.empty(q.shape, dtype=qt, device=DEV)
        ops.prompt_attention(engine, q.to(DEV), k.to(DEV), v.to(DEV), out, 1, n)
        keep = [j for j in range(n) if j != 3]
        want, tol = attend(q, k[keep], v[keep], [r + 1 - (r >= 3) for r in range(n)], qt == torch.float16,
                           kt == torch.float16)
        got = out.float().cpu()
        assert got[17, 1].isnan().all()
        got[17, 1] = want[17, 1] = 0.0
        tol[17, 1] = 1.0
        check(got, want, tol, types)


def _prefix(engine, types, heads, kvh, hd, batch, prefix, lens, cap=None, seed=0, first=3, seq_len=None, device="cpu"):
    qt, kt = TYPES[types]
    gen = torch.Generator().manual_seed(seed)
    cap = cap or max(1, max(lens))
    q = _rand(gen, batch, heads, hd, dtype=qt, sigma=1.5)
    total = first + prefix + batch * cap
    k, v = (_rand(gen, total, kvh, hd, dtype=kt) for _ in range(2))
    slots = torch.randperm(batch, generator=gen).tolist()
    base = [first + prefix + s * cap for s in slots]
    kc, vc = k.clone(), v.clone()
    kc[:first], vc[:first] = math.nan, math.nan
    for b, n in zip(base, lens):
        kc[b + n:b + cap], vc[b + n:b + cap] = math.nan, math.inf
    out = torch.empty(q.shape, dtype=qt, device=DEV)
    ops.prefix_attention(engine, q.to(DEV), kc.to(DEV), vc.to(DEV), out, first, prefix, cap, row_base=_i32(base),
                         seq_lens=_i32(lens) if seq_len is None else None, seq_len=seq_len or 0)
    q, k, v = (x.to(device) for x in (q, k, v))
    with torch.device(device):
        for r, (b, n) in enumerate(zip(base, lens)):
            kk = torch.cat([k[first:first + prefix], k[b:b + n]])
            vv = torch.cat([v[first:first + prefix], v[b:b + n]])
            want, tol = attend(q[r:r + 1], kk, vv, [prefix + n], qt == torch.float16, kt == torch.float16)
            check(out[r:r + 1], want.cpu(), tol.cpu(), (types, r, n))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 65, 1030])
def test_prefix_lengths(engine, types, prefix):
    _prefix(engine, types, 8, 2, 128, 5, prefix, [1, 0, 17, 64, 130])


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("heads,kvh,hd,batch", [(4, 2, 64, 1), (32, 32, 128, 3), (5, 1, 64, 70), (40, 8, 128, 33), (300, 2, 64, 2)])
def test_prefix_batches(engine, types, heads, kvh, hd, batch):
    _prefix(engine, types, heads, kvh, hd, batch, 200, [(i * 37) % 90 for i in range(batch)], cap=100)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_prefix_alone_and_one_length_for_all(engine, types):
    _prefix(engine, types, 8, 2, 64, 4, 300, [0, 0, 0, 0])
    _prefix(engine, types, 8, 2, 64, 4, 300, [21] * 4, cap=32, seq_len=21)
    _prefix(engine, types, 8, 2, 64, 4, 0, [0, 5, 0, 1])
    _prefix(engine, types, 32, 8, 128, 2, 0, [900, 1500])


@pytest.mark.parametrize("types", sorted(TYPES))
def test_more_prefix_and_own_workgroups_than_cus(engine, types):
    _prefix(engine, types, 32, 8, 128, 64, 8300, [(i * 53) % 150 for i in range(64)], cap=150, device=DEV)
    _prefix(engine, types, 16, 8, 64, 130, 4200, [(i * 29) % 40 for i in range(130)], cap=40, device=DEV)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("heads,kvh,rows", [(8, 8, 300), (8, 1, 90), (32, 8, 20)])
def test_long_contexts_in_tiles_of_every_width(engine, types, heads, kvh, rows):
    _prompt(engine, types, heads, kvh, 64, [(rows, 1900)], device=DEV)
    _prompt(engine, types, heads, kvh, 128, [(rows, rows + 700), (1, 650)], device=DEV)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("rows,length", [(1, 2500), (5, 700), (5, 1500), (8, 2500), (12, 1300)])
def test_drafts_behind_long_contexts(engine, types, rows, length):
    # 4 to 48 columns of a sequence in one tile, split or whole; one context shorter than a part
    seqs = [(rows, length), (rows, length // 3), (1, 90), (rows, length - 77), (0, 40), (rows, rows)]
    for hd in (64, 128):
        _prompt(engine, types, 32, 8, hd, seqs, device=DEV)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("nseq", [11, 20])
@pytest.mark.parametrize("hd", [64, 128])
def test_many_tiles_of_many_heads(engine, types, nseq, hd):
    # more tiles than two for each CU: by the position they reach (few sequences on a binary32 cache) or in order
    seqs = [(128, 128), (5, 9), (0, 0), (100, 127), (2, 1), (128, 100)]
    _prompt(engine, types, 32, 32, hd, [seqs[i % 6] if i % 7 else (110 + i % 9, 120) for i in range(nseq)], cap=128, device=DEV)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_split_contexts_of_more_sequences_than_lanes(engine, types):
    _prompt(engine, types, 4, 1, 64, [((i * 5) % 3, (i * 211) % 1500) for i in range(131)], cap=1500, device=DEV)


def test_max_seq_len_without_a_bound(engine):
    """The largest max_seq_len with tables: it only bounds the lengths and plans."""
    gen = torch.Generator().manual_seed(34)
    q = _rand(gen, 3, 8, 64, dtype=torch.float16)
    k, v = (_rand(gen, 900, 2, 64, dtype=torch.float16) for _ in range(2))
    out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
    lens, base = [890, 3, 0], [0, 890, 5]
    for hint in (0, 0xffffffff):
        ops.prompt_attention(engine, q.to(DEV), k.to(DEV), v.to(DEV), out, 3, 0xffffffff, row_base=_i32(base),
                             seq_lens=_i32(lens), max_len_hint=hint)
        for r, (b, n) in enumerate(zip(base, lens)):
            want, tol = attend(q[r:r + 1], k[b:b + n], v[b:b + n], [n], True, True)
            check(out[r:r + 1], want, tol, (hint, r))
        ops.prefix_attention(engine, q.to(DEV), k.to(DEV), v.to(DEV), out, 100, 50, 0xffffffff, row_base=_i32(base),
                             seq_lens=_i32(lens), max_len_hint=hint)
        for r, (b, n) in enumerate(zip(base, lens)):
            kk, vv = (torch.cat([x[100:150], x[b:b + n]]) for x in (k, v))
            want, tol = attend(q[r:r + 1], kk, vv, [50 + n], True, True)
            check(out[r:r + 1], want, tol, (hint, r))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2000), (70, 70), (200, 1400)])
def test_in_place(engine, types, rows, n):
    qt, kt = TYPES[types]
    gen = torch.Generator().manual_seed(31)
    q = _rand(gen, rows, 8, 128, dtype=qt).to(DEV)
    k, v = (_rand(gen, n, 2, 128, dtype=kt).to(DEV) for _ in range(2))
    lens = _i32([n])
    want, got = torch.empty_like(q), q.clone()
    ops.prompt_attention(engine, q, k, v, want, 1, n, seq_lens=lens)
    ops.prompt_attention(engine, got, k, v, got, 1, n, seq_lens=lens)
    assert torch.equal(got, want)
    base, own = _i32([0] * rows), _i32([i % 2 for i in range(rows)])
    got = q.clone()
    ops.prefix_attention(engine, q, k, v, want, 0, n, 1, row_base=base, seq_lens=own)
    ops.prefix_attention(engine, got, k, v, got, 0, n, 1, row_base=base, seq_lens=own)
    assert torch.equal(got, want)


def test_sequences_that_share_cache_rows(engine):
    """The same cache rows under several sequences: every one reads them."""
    gen = torch.Generator().manual_seed(32)
    q = _rand(gen, 6, 8, 64, dtype=torch.float16)
    k, v = (_rand(gen, 90, 2, 64, dtype=torch.float16) for _ in range(2))
    out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
    ops.prompt_attention(engine, q.to(DEV), k.to(DEV), v.to(DEV), out, 3, 90, row_base=_i32([0, 0, 10]),
                         seq_lens=_i32([80, 40, 80]))
    for s, (b, m) in enumerate(((0, 80), (0, 40), (10, 80))):
        want, tol = attend(q[2 * s:2 * s + 2], k[b:b + m], v[b:b + m], [m - 1, m], True, True)
        check(out[2 * s:2 * s + 2], want, tol, s)


def test_two_contexts_at_once(engine):
    """Split calls of two contexts on two streams, many in flight: each has its own
    partials, and every result has the bits of the calls alone."""
    gen = torch.Generator().manual_seed(33)
    heads, kvh, hd, cap = 32, 8, 128, 3000
    k, v = (_rand(gen, 2 * cap, kvh, hd, dtype=torch.float16).to(DEV) for _ in range(2))
    lens, own, base = _i32([cap, 2500]), _i32([300] * 16), _i32([cap + 100 * i for i in range(16)])
    q1, q2 = (_rand(gen, n, heads, hd, dtype=torch.float16).to(DEV) for n in (4, 16))
    engs = [ops.ComputeEngine(0) for _ in range(2)]
    sides = [torch.cuda.Stream() for _ in range(2)]

    def call(eng, which, out):
        if which == 0:
            ops.prompt_attention(eng, q1, k, v, out, 2, cap, seq_lens=lens)
        else:
            ops.prefix_attention(eng, q2, k, v, out, 0, cap, 300, row_base=base, seq_lens=own)

    try:
        torch.cuda.synchronize()
        for eng, side in zip(engs, sides):
            eng.bind_stream(side)
        alone = [torch.empty_like(q1), torch.empty_like(q2)]
        for i in (0, 1):
            call(engs[i], i, alone[i])
            engs[i].sync()
        outs = [[torch.empty_like(alone[i]) for _ in range(20)] for i in (0, 1)]
        torch.cuda.synchronize()
        for j in range(20):
            for i in (0, 1):
                call(engs[i], i, outs[i][j])
        for eng in engs:
            eng.sync()
        for i in (0, 1):
            for j, out in enumerate(outs[i]):
                assert torch.equal(out, alone[i]), (i, j)
    finally:
        for eng in engs:
            eng.sync()
            eng.close()


def test_agrees_with_decode_attention(engine):
    """The same positions through janus_attention, with the prefix copied behind each sequence's base."""
    gen = torch.Generator().manual_seed(9)
    batch, heads, kvh, hd, prefix, cap = 6, 32, 8, 128, 384, 512
    lens = [1, 5, 100, 30, 128, 77]
    q = _rand(gen, batch, heads, hd).to(DEV)
    pk, pv = (_rand(gen, prefix, kvh, hd, dtype=torch.float16).to(DEV) for _ in range(2))
    k, v = (_rand(gen, batch * cap, kvh, hd, dtype=torch.float16).to(DEV) for _ in range(2))
    for s in range(batch):
        k[s * cap:s * cap + prefix], v[s * cap:s * cap + prefix] = pk, pv
    want, got = torch.empty_like(q), torch.empty_like(q)
    ops.compute_attention(engine, q, k, v, want, batch, 0, cap, heads, kvh, hd,
                          seq_lens=_i32([prefix + n for n in lens]))
    ops.prefix_attention(engine, q, k, v, got, 2 * cap, prefix, cap - prefix, seq_lens=_i32(lens),
                         row_base=_i32([s * cap + prefix for s in range(batch)]))
    for s in range(batch):
        _, tol = attend(q[s:s + 1].cpu(), k[s * cap:s * cap + prefix + lens[s]].cpu(),
                        v[s * cap:s * cap + prefix + lens[s]].cpu(), [prefix + lens[s]], False, True)
        check(got[s:s + 1], want[s:s + 1].double().cpu(), 2 * tol, s)


def test_rows_past_32_bits(engine):
    """Cache rows whose byte and element offsets exceed 2^32."""
    heads, kvh, hd, rows = 8, 8, 128, 4_300_000   # 2 KiB a row
    k = torch.empty(rows, kvh, hd, dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    gen = torch.Generator().manual_seed(11)
    kk, vv = (_rand(gen, 300, kvh, hd, dtype=torch.float16) for _ in range(2))
    base = rows - 300
    k[base:], v[base:] = kk.to(DEV), vv.to(DEV)
    q = _rand(gen, 2, heads, hd, dtype=torch.float16)
    out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
    ops.prompt_attention(engine, q.to(DEV), k, v, out, 1, 300, row_base=_i32([base]), seq_lens=_i32([300]))
    want, tol = attend(q, kk, vv, [299, 300], True, True)
    check(out, want, tol)
    ops.prefix_attention(engine, q.to(DEV), k, v, out, base, 200, 100, row_base=_i32([base + 200] * 2), seq_lens=_i32([50, 100]))
    for r, n in ((0, 250), (1, 300)):
        want, tol = attend(q[r:r + 1], kk[:n], vv[:n], [n], True, True)
        check(out[r:r + 1], want, tol, r)


def test_captured_calls_share_the_workspace(engine):
    """Two graphs, both with split partials in the one workspace, replayed in turn
    with eager calls between; lengths and queries change in place."""
    gen = torch.Generator().manual_seed(12)
    heads, kvh, hd, cap = 32, 8, 128, 1200
    k, v = (_rand(gen, 2 * cap, kvh, hd, dtype=torch.float16).to(DEV) for _ in range(2))
    q = _rand(gen, 2, heads, hd, dtype=torch.float16).to(DEV)
    lens, own = _i32([cap, 700]), _i32([3, 5])
    base = _i32([600, 1500])
    out1, out2 = torch.empty_like(q), torch.empty_like(q)
    side = torch.cuda.Stream()
    eng = ops.ComputeEngine(0)
    try:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eng.bind_stream()
            def prompt(out):
                ops.prompt_attention(eng, q, k, v, out, 2, cap, seq_lens=lens)
            def prefix(out):
                ops.prefix_attention(eng, q, k, v, out, 0, 600, 8, row_base=base, seq_lens=own)
            prompt(out1), prefix(out2)   # the workspace grows outside the captures
            side.synchronize()
            g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
            with torch.cuda.graph(g1, stream=side):
                eng.bind_stream(side)
                prompt(out1)
            with torch.cuda.graph(g2, stream=side):
                prefix(out2)
            for i in range(4):
                lens.copy_(_i32([cap - 100 * i, 700 + i]))
                own.copy_(_i32([i, 8 - i]))
                q.copy_(_rand(gen, 2, heads, hd, dtype=torch.float16))
                out1.zero_(), out2.zero_()
                g1.replay(), g2.replay(), g1.replay()
                e1, e2 = torch.empty_like(q), torch.empty_like(q)
                prompt(e1), prefix(e2)
                side.synchronize()
                assert torch.equal(out1, e1) and torch.equal(out2, e2), i
    finally:
        eng.sync()
        eng.close()


def test_growth_inside_a_capture_is_refused():
    eng = ops.ComputeEngine(0)
    side = torch.cuda.Stream()
    k = torch.zeros(4096, 8, 128, dtype=torch.float16, device=DEV)
    q = torch.zeros(64, 32, 128, dtype=torch.float16, device=DEV)
    lens, out = _i32([4096] * 64), torch.zeros_like(q)
    base = _i32([0] * 64)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        eng.bind_stream(side)
        out.zero_()
        with pytest.raises(ops.JanusError, match="reserve it before capturing"):
            ops.prefix_attention(eng, q, k, k, out, 0, 4096, 4096, row_base=base, seq_lens=lens)
    torch.cuda.synchronize()
    eng.close()


def test_another_stream_and_repeated_calls_give_the_same_bits(engine):
    gen = torch.Generator().manual_seed(13)
    q = _rand(gen, 300, 8, 128, dtype=torch.float16).to(DEV)
    k, v = (_rand(gen, 600, 2, 128, dtype=torch.float16).to(DEV) for _ in range(2))
    a, b = torch.empty_like(q), torch.empty_like(q)
    torch.cuda.synchronize()
    ops.prompt_attention(engine, q, k, v, a, 1, 600, seq_lens=_i32([600]))
    engine.sync()
    side = torch.cuda.Stream()
    eng = ops.ComputeEngine(0)
    lens = _i32([600])
    torch.cuda.synchronize()
    eng.bind_stream(side)
    ops.prompt_attention(eng, q, k, v, b, 1, 600, seq_lens=lens)
    eng.sync()
    assert torch.equal(a, b)
    eng.close()
