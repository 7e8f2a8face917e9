"""Tables of janus_fp4_attention at the ends of what they may hold."""
import pytest
import torch

from janus_amd import ops
from fp4_ref import decode, random_cache
from packed_ref import attend, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("rows", [1, 9, 40])
@pytest.mark.parametrize("cap", [50, 1500])
def test_the_longest_length_without_rows(engine, rows, cap):
    """A sequence without rows whose length is the largest there is, between others; one with rows and that length."""
    gen = torch.Generator().manual_seed(61)
    heads, kvh, hd = 8, 4, 128
    cache = [*random_cache(gen, 3 * cap, kvh, hd), *random_cache(gen, 3 * cap, kvh, hd)]
    k, v = decode(*cache[:2]), decode(*cache[2:])
    q = torch.randn(2 * rows, heads, hd, generator=gen).half()
    out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
    big = 2 ** 31 - 1
    ops.fp4_attention(engine, q.to(DEV), *[c.to(DEV) for c in cache], out, 4, cap, q_start=_i32([0, 0, rows, rows, 2 * rows]),
                      row_base=_i32([0, cap, 0, 2 * cap]), seq_lens=_i32([big, cap, big, big]))
    for s, base, seen in ((0, cap, [cap - rows + 1 + r for r in range(rows)]), (1, 2 * cap, [cap] * rows)):
        at, on = slice(s * rows, (s + 1) * rows), slice(base, base + cap)
        want, tol = attend(q[at], k[on], v[on], seen, True, True)
        check(out[at], want, tol, (rows, cap, s))
