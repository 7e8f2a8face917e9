"""Weights of janus_prompt_attention whose exponents leave 32 bits."""
import math

import pytest
import torch

from janus_amd import ops
from packed_ref import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f16_f16": (torch.float16, torch.float16), "f32_f16": (torch.float32, torch.float16),
         "f32_f32": (torch.float32, torch.float32)}


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("rows,heads,kvh,n", [(3, 4, 2, 1100), (20, 8, 8, 300), (40, 8, 2, 90), (70, 8, 8, 1100), (150, 64, 32, 150)])
@pytest.mark.parametrize("hd", [64, 128])
def test_scores_far_below_zero(engine, types, rows, heads, kvh, n, hd):
    """Every score is below -2^128 in powers of two, beyond binary32, though q, K and the scale are finite: the sums
    q k are whole multiples of the size of q, exact in binary32, and what is not equal to the largest has no weight."""
    gen = torch.Generator().manual_seed(53)
    rt, ct = TYPES[types]
    size, scale = (2.0 ** 14, 2.0 ** 113) if rt == torch.float16 else (2.0 ** 115, 2.0 ** 10)
    q = torch.full((rows, heads, hd), size, dtype=rt)
    k = torch.where(torch.rand(n, kvh, hd, generator=gen) < 0.5, -4.0, -3.0).to(ct)
    v = torch.randn(n, kvh, hd, generator=gen).to(ct)
    out = torch.empty(rows, heads, hd, dtype=rt, device=DEV)
    ops.prompt_attention(engine, q.to(DEV), k.to(DEV), v.to(DEV), out, 1, n,
                         seq_lens=torch.tensor([n], dtype=torch.int32, device=DEV), scale=scale)
    seen = torch.arange(n)[None] < torch.arange(n - rows + 1, n + 1)[:, None]
    for h in range(heads):
        s = (q[:, h].double() @ k[:, h // (heads // kvh)].double().T).masked_fill(~seen, -math.inf)
        assert s.max() * scale * math.log2(math.e) < -2.0 ** 128
        first = (s == s.amax(-1, keepdim=True)).double()
        vh = v[:, h // (heads // kvh)].double()
        want = first @ vh / first.sum(-1, keepdim=True)
        tol = 2.0 ** (-10 if rt == torch.float16 else -20) * vh.abs().max()
        check(out[:, h], want, tol.expand_as(want), (types, h))
