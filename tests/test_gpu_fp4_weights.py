"""Weights of janus_fp4_attention whose exponents meet the limits of 32 bits."""
import math

import pytest
import torch

from janus_amd import ops
from fp4_ref import decode, random_cache
from packed_ref import U32, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f16": torch.float16, "f32": torch.float32}


def _attend(engine, q, cache, n, scale, nseq=1):
    out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
    ops.fp4_attention(engine, q.to(DEV), *[c.to(DEV) for c in cache], out, nseq, n,
                      seq_lens=torch.full((nseq,), n, dtype=torch.int32, device=DEV), scale=scale)
    return out.cpu()


def _the_best_share(got, q, k, v, types):
    """Scores so far apart that the largest of what a row sees takes all weight, equal ones share it."""
    rows, heads, _ = q.shape
    n, rep = k.shape[0], heads // k.shape[1]
    seen = torch.arange(n)[None] < torch.arange(n - rows + 1, n + 1)[:, None]
    for h in range(heads):
        s = (q[:, h].double() @ k[:, h // rep].T).masked_fill(~seen, -math.inf)
        first = (s == s.amax(-1, keepdim=True)).double()
        want = first @ v[:, h // rep] / first.sum(-1, keepdim=True)
        tol = 2.0 ** (-10 if types == "f16" else -20) * v.abs().max()
        check(got[:, h], want, tol.expand_as(want), (types, h))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("rows,heads,kvh,n", [(3, 4, 2, 1100), (20, 8, 8, 300), (70, 8, 8, 1100), (40, 8, 2, 90)])
def test_scores_far_below_zero(engine, types, rows, heads, kvh, n):
    """Every score is below -2^128 in powers of two, beyond binary32, though q, K and the scale are finite: the sums
    q k are whole multiples of the size of q, exact in binary32, and what is not equal to the largest has no weight."""
    gen = torch.Generator().manual_seed(51)
    size, scale = (2.0 ** 14, 2.0 ** 112) if types == "f16" else (2.0 ** 122, 2.0)
    q = torch.full((rows, heads, 128), size, dtype=TYPES[types])
    codes = torch.where(torch.rand(n, kvh, 64, generator=gen) < 0.5, 0xEE, 0xDE).to(torch.uint8)   # -4, or -4 and -3
    cache = [codes, torch.full((n, kvh, 4), 127, dtype=torch.uint8), *random_cache(gen, n, kvh, 128)]
    k, v = decode(*cache[:2]), decode(*cache[2:])
    assert (q[:1, :kvh].double() * k).sum(-1).max() * scale * math.log2(math.e) < -2.0 ** 128
    _the_best_share(_attend(engine, q, cache, n, scale), q, k, v, types)


def test_scores_far_below_zero_of_many_tiles(engine):
    """As above, 32 KV heads of 140 columns, 4 sequences."""
    gen = torch.Generator().manual_seed(52)
    n, kvh = 70, 32
    q = torch.full((4 * n, 2 * kvh, 128), 2.0 ** 14, dtype=torch.float16)
    codes = torch.where(torch.rand(4 * n, kvh, 64, generator=gen) < 0.5, 0xEE, 0xDE).to(torch.uint8)
    cache = [codes, torch.full((4 * n, kvh, 4), 127, dtype=torch.uint8), *random_cache(gen, 4 * n, kvh, 128)]
    k, v = decode(*cache[:2]), decode(*cache[2:])
    got = _attend(engine, q, cache, n, 2.0 ** 112, nseq=4)
    for s in range(4):
        at = slice(s * n, (s + 1) * n)
        _the_best_share(got[at], q[at], k[at], v[at], "f16")


def _unit_keys(n, kvh, at):
    """Codes and scales of K: 1 in the dims that `at` names for a position, else 0."""
    codes = torch.zeros(n, kvh, 64, dtype=torch.uint8)
    for p, dims in at.items():
        for d in dims:
            codes[p, :, d // 2] |= 2 << 4 * (d % 2)
    return [codes, torch.full((n, kvh, 4), 127, dtype=torch.uint8)]


@pytest.mark.parametrize("rows", [3, 20, 60])
def test_a_maximum_that_goes_beyond_2_to_22(engine, rows):
    """The running maximum, in powers of two, is 4194311.17 and later 4194318.38: on this way kBias less its offset
    (-4194298.25) is not a binary32 number, the next ones are 1/4 away. The scores are exact, and the weight of the
    first position is e^-5."""
    a, later, n, kvh = 2907275, 5, 70 + rows, 8
    q = torch.zeros(rows, kvh, 128)
    q[..., 0], q[..., 1] = a, later
    cache = _unit_keys(n, kvh, {0: [0], 64: [0, 1]}) + [*random_cache(torch.Generator().manual_seed(54), n, kvh, 128)]
    v = decode(*cache[2:])
    w = math.exp(-later)
    want = ((v[64] + w * v[0]) / (1 + w)).expand(rows, kvh, 128)
    # scale log2(e) is rounded (2 u of 5 log2(e)), the weight by 2^-22, each step of the joined sums by u
    tol = w * (10 * 1.45 * U32 + 2.0 ** -22) * (v[64] - v[0]).abs() + 8 * U32 * (v[64].abs() + v[0].abs())
    check(_attend(engine, q, cache, n, 1.0), want, tol.expand(rows, kvh, 128), rows)


@pytest.mark.parametrize("rows", [3, 20, 60])
@pytest.mark.parametrize("a,b", [(9.483467102050781, 9.483417510986328), (8.494361877441406, 8.49441146850586),
                                 (2907272, 2907273), (2907274, 2907275)])
def test_parts_are_joined_by_what_their_weights_mean(engine, rows, a, b):
    """Positions 0 to 31 of 64 have the score a, the others b, which one wavefront, or one of a pair each, takes: both
    are exact, but kBias less their offsets rounds to either side, by 2^-21 (1/4) in powers of two. With V of 1 and -1 the
    output is (A - B) / (A + B), off by half the difference of the weights' errors of up to 2^-22 each."""
    n, kvh = 64, 8
    q = torch.zeros(rows, kvh, 128)
    q[..., 0], q[..., 1] = a, b
    cache = _unit_keys(n, kvh, {p: [0 if p < 32 else 1] for p in range(n)})
    sign = torch.where(torch.arange(n) < 32, 0x22, 0xAA).to(torch.uint8)
    cache += [sign[:, None, None].expand(n, kvh, 64).contiguous(), torch.full((n, kvh, 4), 127, dtype=torch.uint8)]
    seen = torch.arange(n - rows + 1, n + 1).double()
    one, two = seen.clamp(max=32), (seen - 32).clamp(min=0) * math.exp(b - a)
    want = ((one - two) / (one + two))[:, None, None].expand(rows, kvh, 128)
    tol = 2.0 ** -22 + 8 * U32 * want.abs() + 2 * 1.45 * U32 * abs(b - a)
    check(_attend(engine, q, cache, n, 1.0), want, tol, (rows, a, b))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("rows,n", [(3, 200), (20, 200), (60, 1500)])
def test_factors_beyond_32_bits(engine, types, rows, n):
    """log2(e) times the scale, or that times a row's power of two, is above the largest binary32 number: what is
    not equal to the largest score has no weight."""
    gen = torch.Generator().manual_seed(55)
    kvh = 8
    size, scale = (1.0, 3e38) if types == "f16" else (2.0 ** 126, 2.0 ** 20)
    q = torch.full((rows, kvh, 128), size, dtype=TYPES[types])
    codes = torch.where(torch.rand(n, kvh, 64, generator=gen) < 0.5, 0x22, 0xA2).to(torch.uint8)   # 1, or 1 and -1
    cache = [codes, torch.full((n, kvh, 4), 127, dtype=torch.uint8), *random_cache(gen, n, kvh, 128)]
    _the_best_share(_attend(engine, q, cache, n, scale), q, decode(*cache[:2]), decode(*cache[2:]), types)
