"""Infinities, NaN and extreme scores where the attentions of packed rows share K
and V through LDS: many columns, in one piece (PACKED: with binary16 rows and 128
dims three workgroups on a CU, else two) and in parts (SPLIT), and behind a prefix."""
import math

import pytest
import torch

from janus_amd import ops
from packed_ref import attend, check
from test_gpu_packed_attention import DEV, TYPES, _i32, _prompt, _rand

pytestmark = pytest.mark.gpu

# 128 columns of a sequence and head, 640 and more tiles: never split, never narrow
PACKED = [(120 + 5 * (i % 4), 120 + 5 * (i % 4) + (0, 0, 37, 300)[i % 4]) for i in range(20)]
# 160 and 280 columns of a KV head behind contexts that take several workgroups
SPLIT = [(40, 3000), (70, 2211)]
SHAPES = {"packed": (32, 32, PACKED), "split": (32, 8, SPLIT)}


def _place(q, k, v, p, group):
    """Odd values at position p of K and V [len, kv heads, hd], one kind per KV head:
      0: +infinity in V, dim 5, and -infinity in dim 6 a position later;
      1: NaN in V, dim 7;     2: NaN in K;      3: +infinity in K, where q > 0;
      4: -infinity in K, where q > 0: a position without weight;
      5: a NaN row of q (the last but one), and an infinite one (the last)."""
    v[p, 0, 5], v[p + 1, 0, 6], v[p, 1, 7] = math.inf, -math.inf, math.nan
    k[p, 2, 3] = math.nan
    for h, x in ((3, math.inf), (4, -math.inf)):
        q[:, h * group:(h + 1) * group, 9] = q[:, h * group:(h + 1) * group, 9].abs() + 0.5
        k[p, h, 9] = x
    q[-2, 5 * group, 11], q[-1, 6 * group - 1, 12] = math.nan, math.inf


def _check_odd(got, q, k, v, seen, p, group, types, what):
    """got [n, heads, hd]; row r of q sees the first seen[r] positions of K and V,
    which hold the values of _place at position p (None: they do not)."""
    got, seen = got.double().cpu(), torch.as_tensor(seen)
    sees, later = (seen > p, seen > p + 1) if p is not None else (seen < 0, seen < 0)
    heads = [slice(h * group, (h + 1) * group) for h in range(k.shape[1])]
    lost = torch.zeros(got.shape, dtype=torch.bool)   # NaN expected
    lost[sees, heads[1], 7], lost[sees, heads[2]], lost[sees, heads[3]] = True, True, True
    lost |= ~q.isfinite().all(-1, keepdim=True)
    assert got[lost].isnan().all(), what
    assert (got[sees, heads[0], 5] == math.inf).all() and (got[later, heads[0], 6] == -math.inf).all(), what
    lost[sees, heads[0], 5], lost[later, heads[0], 6] = True, True
    q, k, v = (x.nan_to_num(0.0, 0.0, 0.0).to(DEV) for x in (q, k, v))
    want, tol = torch.zeros(got.shape, dtype=torch.float64), torch.zeros(got.shape, dtype=torch.float64)
    for h, part in enumerate(heads):
        gone = h == 4 and p is not None
        keep = [j for j in range(k.shape[0]) if not gone or j != p]
        with torch.device(DEV):
            w, t = attend(q[:, part], k[keep, h:h + 1], v[keep, h:h + 1], (seen - sees.long() * gone).tolist(),
                          *(x == torch.float16 for x in TYPES[types]))
        want[:, part], tol[:, part] = w.cpu(), t.cpu()
    check(torch.where(lost, 0.0, got), torch.where(lost, 0.0, want), tol + lost, what)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("hd", [64, 128])
def test_odd_values(engine, types, shape, hd):
    """Two sequences hold odd values, one among its last rows' own positions (rows
    before them see none of it) and one in its context; the others hold none. What
    lies behind a sequence is NaN and infinite. In place gives the same bits."""
    heads, kvh, seqs = SHAPES[shape]
    qt, kt = TYPES[types]
    gen = torch.Generator().manual_seed(51)
    group, cap = heads // kvh, max(m for _, m in seqs) + 3
    odd = {0: 77, 3: 100} if shape == "packed" else {0: 2985, 1: 1000}
    data, starts = [], [0]
    kc = torch.full((len(seqs) * cap, kvh, hd), math.nan, dtype=kt)
    vc = torch.full_like(kc, math.inf)
    for s, (n, m) in enumerate(seqs):
        q, k, v = _rand(gen, n, heads, hd, dtype=qt), *(_rand(gen, m, kvh, hd, dtype=kt) for _ in range(2))
        if s in odd:
            _place(q, k, v, odd[s], group)
        kc[s * cap:s * cap + m], vc[s * cap:s * cap + m] = k, v
        data.append((q, k, v))
        starts.append(starts[-1] + n)
    q = torch.cat([x[0] for x in data]).to(DEV)
    out = torch.empty_like(q)
    kc, vc, lens, base = kc.to(DEV), vc.to(DEV), _i32([m for _, m in seqs]), _i32([s * cap for s in range(len(seqs))])
    ops.prompt_attention(engine, q, kc, vc, out, len(seqs), cap, q_start=_i32(starts), row_base=base, seq_lens=lens)
    got = out.cpu()
    for s, (n, m) in enumerate(seqs):
        mine, seen = got[starts[s]:starts[s + 1]], [m - n + 1 + r for r in range(n)]
        if s in odd or s in (1, 2, 19):
            _check_odd(mine, *data[s], seen, odd.get(s), group, types, (types, s))
        else:
            assert mine.isfinite().all(), s
    ops.prompt_attention(engine, q, kc, vc, q, len(seqs), cap, q_start=_i32(starts), row_base=base, seq_lens=lens)
    same = (q == out) | (q.isnan() & out.isnan())
    assert same.all()


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_odd_values_behind_a_prefix(engine, types, where):
    """64 requests behind 4100 shared positions (128 columns a workgroup): the odd
    values of the prefix reach all of them, those of a request that request alone."""
    heads, kvh, hd, batch, prefix, cap = 32, 8, 128, 64, 4100, 40
    qt, kt = TYPES[types]
    gen = torch.Generator().manual_seed(52)
    q = _rand(gen, batch, heads, hd, dtype=qt)
    k, v = (_rand(gen, prefix + batch * cap, kvh, hd, dtype=kt) for _ in range(2))
    lens = [20 + i % 21 for i in range(batch)]
    odd = 1234 if where == "prefix" else prefix + 8 * cap + 7
    _place(q, k, v, odd, heads // kvh)
    out = torch.empty_like(q, device=DEV)
    ops.prefix_attention(engine, q.to(DEV), k.to(DEV), v.to(DEV), out, 0, prefix, cap,
                         row_base=_i32([prefix + s * cap for s in range(batch)]), seq_lens=_i32(lens))
    got = out.cpu()
    for s in (0, 8, 33, 62, 63):
        at = list(range(prefix)) + list(range(prefix + s * cap, prefix + s * cap + lens[s]))
        p = at.index(odd) if odd in at else None
        _check_odd(got[s:s + 1], q[s:s + 1], k[at], v[at], [len(at)], p, heads // kvh, types, (types, s))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("sigma", [0.0, 1e-6, 40.0])
def test_score_ranges(engine, types, shape, sigma):
    heads, kvh, seqs = SHAPES[shape]
    _prompt(engine, types, heads, kvh, 128, seqs, sigma=sigma, device=DEV)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_scores_beyond_their_own_last_bits(engine, types, shape):
    """Scores whose spacing is far above 1: the farthest ahead takes all weight, equal
    ones share it. (Weights and their sums are whole numbers, the quotient and the
    products with v are rounded: far below the bound's 4 steps of the output's type.)"""
    heads, kvh, seqs = SHAPES[shape]
    qt, kt = TYPES[types]
    gen = torch.Generator().manual_seed(53)
    hd, cap = 128, max(m for _, m in seqs)
    size = 3e4 if qt == torch.float16 else 3.0 * 2 ** 25   # products and sums are exact
    q = (_rand(gen, sum(n for n, _ in seqs), heads, hd).sign() * size).to(qt)
    k = (_rand(gen, len(seqs) * cap, kvh, hd).sign() * 64).to(kt)
    v = _rand(gen, len(seqs) * cap, kvh, hd, dtype=kt)
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    out = torch.empty(q.shape, dtype=qt, device=DEV)
    ops.prompt_attention(engine, q.to(DEV), k.to(DEV), v.to(DEV), out, len(seqs), cap, q_start=_i32(starts),
                         seq_lens=_i32([m for _, m in seqs]))
    got, group = out.double().cpu(), heads // kvh
    tol = 2.0 ** (-10 if qt == torch.float16 else -20) * v.abs().max().double()
    for s, (n, m) in list(enumerate(seqs))[:4]:
        there = torch.arange(m)[None] < (m - n + 1 + torch.arange(n))[:, None]
        for h in range(0, heads, 5):
            at = slice(s * cap, s * cap + m)
            score = q[starts[s]:starts[s + 1], h].double() @ k[at, h // group].double().T
            score = score.masked_fill(~there, -math.inf)
            first = (score == score.amax(-1, keepdim=True)).double()
            want = first @ v[at, h // group].double() / first.sum(-1, keepdim=True)
            check(got[starts[s]:starts[s + 1], h], want, tol.expand_as(want), (types, s, h))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_rising_scores(engine, types, shape):
    # the maximum moves with every tile: each rescales what came before
    heads, kvh, seqs = SHAPES[shape]
    qt, kt = TYPES[types]
    f16 = qt == torch.float16, kt == torch.float16
    hd, cap = 128, max(m for _, m in seqs)
    rows = sum(n for n, _ in seqs)
    q = torch.ones(rows, heads, hd, dtype=qt)
    k = (torch.arange(cap)[:, None, None] / 16.0).expand(cap, kvh, hd).to(kt).contiguous()
    v = _rand(torch.Generator().manual_seed(54), cap, kvh, hd, dtype=kt)
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    out = torch.empty(q.shape, dtype=qt, device=DEV)
    ops.prompt_attention(engine, q.to(DEV), k.to(DEV), v.to(DEV), out, len(seqs), cap, q_start=_i32(starts),
                         row_base=_i32([0] * len(seqs)), seq_lens=_i32([m for _, m in seqs]), scale=0.05)
    for s, (n, m) in list(enumerate(seqs))[:4]:
        with torch.device(DEV):
            want, tol = attend(*(x.to(DEV) for x in (q[:n], k[:m], v[:m])), [m - n + 1 + r for r in range(n)], *f16, 0.05)
        check(out[starts[s]:starts[s + 1]], want.cpu(), tol.cpu(), (types, s))


def _least_us(call):
    """Least time of a call over three runs of ten."""
    times = []
    for _ in range(4):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        for _ in range(10):
            call()
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end) * 100)
    return min(times[1:])


def _costs(engine, types, heads, kvh, seqs, most):
    """One odd value of q, K or V, and scores of any size, take at most `most` times
    as long as values without any."""
    qt, kt = TYPES[types]
    gen = torch.Generator(device=DEV).manual_seed(55)
    cap = max(m for _, m in seqs)
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], heads, 128, generator=gen, device=DEV).to(qt)
    k, v = (torch.randn(len(seqs) * cap, kvh, 128, generator=gen, device=DEV).to(kt) for _ in range(2))
    tables = dict(q_start=_i32(starts), seq_lens=_i32([m for _, m in seqs]))
    out = torch.empty_like(q)

    def took():
        return _least_us(lambda: ops.prompt_attention(engine, q, k, v, out, len(seqs), cap, **tables))

    clean = took()
    for t, value in ((v, math.inf), (v, math.nan), (k, math.nan), (k, -math.inf), (q, math.inf), (q, math.nan)):
        was = t[0, :, 3].clone()
        t[0, :, 3] = value
        assert took() <= most * clean, (types, value, clean)
        t[0, :, 3] = was
    q *= 3e4 / q.abs().max().item() if qt == torch.float16 else 1e8
    assert took() <= most * clean, (types, "large", clean)


@pytest.mark.parametrize("types", ["f32", "f32_f16"])
def test_odd_values_cost_little_on_few_columns(engine, types):
    _costs(engine, types, 32, 8, [(5, 1005)] * 16, 4)


@pytest.mark.parametrize("types", ["f16", "f32_f16"])
@pytest.mark.parametrize("heads,kvh,seqs", [(32, 8, [(2048, 2048)]), (32, 8, [(5, 1005)] * 16), (32, 8, SPLIT), (32, 32, PACKED)])
def test_odd_values_cost_little_on_many_columns(engine, types, heads, kvh, seqs):
    # every tile of columns may be computed a second time, at a third to a fifth of the rate
    _costs(engine, types, heads, kvh, seqs, 12)
