"""Attentions of packed rows whose sequences are longer than their cache slots."""
import pytest
import torch

from janus_amd import ops
from packed_ref import attend, check
from test_gpu_packed_attention import DEV, TYPES, _i32, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("heads,kvh,cap,seqs,given", [
    (8, 2, 64, [(100, 100), (10, 10), (64, 64), (65, 65)], False),     # whole prompts, the slots hold 64 positions
    (8, 2, 64, [(50, 100), (3, 64), (5, 66), (70, 140), (1, 90)], True),
    (32, 32, 100, [(120 + i % 9, 120 + i % 9) for i in range(20)], False),   # many columns, tiles by position
    (32, 8, 2980, [(40, 3000), (1, 2981), (30, 2990), (30, 2980)], True)])   # split
def test_sequences_longer_than_their_slots(engine, types, heads, kvh, cap, seqs, given):
    """Rows keep their positions: those whose positions fit see what they see in a
    longer slot, the others all of the slot."""
    qt, kt = TYPES[types]
    gen = torch.Generator().manual_seed(61)
    starts = [0]
    for n, _ in seqs:
        starts.append(starts[-1] + n)
    q = _rand(gen, starts[-1], heads, 128, dtype=qt).to(DEV)
    k, v = (_rand(gen, len(seqs) * cap, kvh, 128, dtype=kt).to(DEV) for _ in range(2))
    out = torch.empty_like(q)
    ops.prompt_attention(engine, q, k, v, out, len(seqs), cap, q_start=_i32(starts),
                         seq_lens=_i32([m for _, m in seqs]) if given else None)
    for s, (n, m) in enumerate(seqs):
        seen = [min(m - n + 1 + r, cap) for r in range(n)]
        with torch.device(DEV):
            want, tol = attend(q[starts[s]:starts[s + 1]], k[s * cap:(s + 1) * cap], v[s * cap:(s + 1) * cap], seen,
                               qt == torch.float16, kt == torch.float16)
        check(out[starts[s]:starts[s + 1]], want.cpu(), tol.cpu(), (types, s, n, m))
