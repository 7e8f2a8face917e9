"""janus_qk_norm_rope against 64 bits, and the operators of packed rows in the
order in which a request meets them."""
import math

import pytest
import torch

from janus_amd import ops
from packed_ref import U16, U32, attend, check, normed_rotated

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
EPS = 1e-5


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _table(n, hd):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    return torch.stack([ang.cos(), ang.sin()], -1).float()


def _heads(engine, rows, heads, kvh, hd, types=(F32, F32, F16), gains=(True, True), base=None, pos=None, cap=40,
           cache_rows=None, fused=True, shift=0, in_place=False, seed=0, sigma=2.0, position=0):
    it, ot, kt = types
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, heads + 2 * kvh, hd, generator=gen) * sigma).to(it)
    dev = torch.empty(x.numel() + shift, dtype=it, device=DEV)[shift:].view(x.shape)
    dev.copy_(x)
    parts = dev.split([heads, kvh, kvh], 1)
    if not fused:
        parts = [p.contiguous() for p in parts]
    gq, gk = ((1 + 0.3 * torch.randn(hd, generator=gen)) if g else None for g in gains)
    table = _table(cap, hd)
    total = cache_rows or (rows * cap if base is None else max(base) + cap)
    kc = torch.full((total, kvh, hd), 3.0, dtype=kt, device=DEV)
    vc = torch.full_like(kc, 3.0)
    out = parts[0] if in_place else torch.full((rows, heads, hd), 7.0, dtype=ot, device=DEV)
    ops.qk_norm_rope(engine, *parts, None if gq is None else gq.to(DEV), None if gk is None else gk.to(DEV), EPS,
                     table.to(DEV), out, kc, vc, cap, position=position,
                     row_base=None if base is None else _i32(base), positions=None if pos is None else _i32(pos))
    engine.sync()
    p = [position] * rows if pos is None else pos
    b = [r * cap for r in range(rows)] if base is None else base
    turns = [r for r in range(rows) if 0 <= p[r] < cap]
    cs = table[[p[r] for r in turns]]
    want, tol = normed_rotated(x[turns, :heads], gq, cs, EPS, ot == F16)
    check(out[turns], want, tol, "q")
    left = [r for r in range(rows) if r not in turns]
    assert in_place or (out[left] == 7.0).all()
    want, tol = normed_rotated(x[turns, heads:heads + kvh], gk, cs, EPS, kt == F16)
    rest = torch.ones(total, dtype=torch.bool)
    for i, r in enumerate(turns):
        if b[r] < 0:
            continue
        at = b[r] + p[r]
        rest[at] = False
        check(kc[at], want[i], tol[i], ("k", r))
        assert torch.equal(vc[at].cpu(), x[r, heads + kvh:].to(kt)), r
    assert (kc[rest.to(DEV)] == 3.0).all() and (vc[rest.to(DEV)] == 3.0).all()


@pytest.mark.parametrize("types", [(F32, F32, F16), (F32, F32, F32), (F32, F16, F16), (F16, F16, F16), (F16, F32, F32),
                                   (F16, F16, F32)])
@pytest.mark.parametrize("heads,kvh,hd", [(4, 2, 64), (32, 8, 128), (3, 1, 256), (2, 2, 96), (5, 1, 2), (1, 1, 1024)])
def test_types_and_head_dims(engine, types, heads, kvh, hd):
    _heads(engine, 7, heads, kvh, hd, types, pos=[0, 5, 39, 1, 2, 3, 4])


@pytest.mark.parametrize("gains", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("hd", [64, 96])
def test_without_a_norm(engine, gains, hd):
    _heads(engine, 5, 4, 2, hd, gains=gains, pos=[3, 1, 4, 1, 5])


@pytest.mark.parametrize("rows", [1, 2, 63, 700, 3001])
@pytest.mark.parametrize("types", [(F32, F32, F16), (F16, F16, F16)])
def test_row_counts(engine, rows, types):
    # a prompt in one slot: consecutive positions; enough rows for both launch shapes
    _heads(engine, rows, 8, 2, 128, types, base=[17] * rows, pos=list(range(rows)), cap=rows + 1)


def test_rows_left_out_and_padding(engine):
    for hd in (64, 96):
        # positions outside the table; negative row bases append nothing
        _heads(engine, 6, 4, 2, hd, base=[0, 40, -1, 80, -5, 120], pos=[-1, 40, 3, 39, 1000000, 0], cap=40)


def test_shared_position(engine):
    _heads(engine, 3, 4, 2, 128, position=11)


@pytest.mark.parametrize("types", [(F32, F32, F16), (F16, F16, F16)])
def test_buffers_that_are_not_aligned(engine, types):
    _heads(engine, 5, 4, 2, 128, types, pos=[3, 1, 4, 1, 5], shift=1)
    _heads(engine, 5, 4, 2, 128, types, pos=[3, 1, 4, 1, 5], shift=1, fused=False)


@pytest.mark.parametrize("types", [(F32, F32, F16), (F16, F16, F16)])
@pytest.mark.parametrize("hd", [64, 96])
def test_in_place(engine, types, hd):
    _heads(engine, 9, 4, 2, hd, types, pos=list(range(9)), fused=False, in_place=True)


def test_zero_and_small_heads(engine):
    # x of 0: eps alone under the root; x below it
    _heads(engine, 4, 4, 2, 64, pos=[1, 2, 3, 4], sigma=0.0)
    _heads(engine, 4, 4, 2, 64, pos=[1, 2, 3, 4], sigma=1e-4)


def test_cache_rows_past_32_bits(engine):
    rows, kvh, hd = 4_300_000, 8, 128
    kc = torch.empty(rows, kvh, hd, dtype=F16, device=DEV)
    vc = torch.empty_like(kc)
    x = torch.randn(2, 8, hd, generator=torch.Generator().manual_seed(2))
    xd = x.to(DEV)
    out = torch.empty_like(xd)
    table = _table(16, hd)
    ops.qk_norm_rope(engine, xd, xd, xd, None, None, EPS, table.to(DEV), out, kc, vc, 16,
                     row_base=_i32([rows - 16, rows - 16]), positions=_i32([15, 3]))
    want, tol = normed_rotated(x, None, table[[15, 3]], EPS, True)
    check(kc[rows - 1], want[0], tol[0])
    check(kc[rows - 13], want[1], tol[1])
    assert torch.equal(vc[rows - 1].cpu(), x[0].half())


def test_captured_call_follows_its_tables(engine):
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(3, 12, 128, generator=gen)
    xd = x.to(DEV)
    table = _table(64, 128).to(DEV)
    kc, vc = (torch.zeros(3 * 64, 2, 128, dtype=F16, device=DEV) for _ in range(2))
    out, pos, base = torch.zeros(3, 8, 128, device=DEV), _i32([0, 1, 2]), _i32([0, 64, 128])
    eng, side = ops.ComputeEngine(0), torch.cuda.Stream()
    q, k, v = xd.split([8, 2, 2], 1)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        eng.bind_stream(side)
        ops.qk_norm_rope(eng, q, k, v, None, None, EPS, table, out, kc, vc, 64, row_base=base, positions=pos)
    for step in range(4):
        with torch.cuda.stream(side):
            pos.add_(5)
            g.replay()
        side.synchronize()
        p = pos.tolist()
        want, tol = normed_rotated(x[:, :8], None, table.cpu()[p], EPS, False)
        check(out, want, tol, step)
        want, tol = normed_rotated(x[:, 8:10], None, table.cpu()[p], EPS, True)
        check(kc[[b + i for b, i in zip(base.tolist(), p)]], want, tol, step)
    eng.close()


@pytest.mark.parametrize("rt,kt", [(F32, F32), (F32, F16), (F16, F16)])
def test_prompts_and_steps_behind_a_shared_prefix(engine, rt, kt):
    """A shared prompt and two requests' own prompts run packed through
    qk_norm_rope and prompt_attention, then two decode steps through qk_norm_rope
    and prefix_attention. Each result is checked against 64 bits on the cache as
    it is, and the cache against 64 bits on the rows."""
    gen = torch.Generator().manual_seed(8)
    heads, kvh, hd, cap, prefix = 8, 2, 128, 48, 150
    total = prefix + 2 * cap
    table = _table(256, hd)
    td = table.to(DEV)
    gq, gk = (1 + 0.3 * torch.randn(hd, generator=gen) for _ in range(2))
    gqd, gkd = gq.to(DEV), gk.to(DEV)
    kc, vc = (torch.zeros(total, kvh, hd, dtype=kt, device=DEV) for _ in range(2))
    f16 = rt == F16, kt == F16

    def rows(n):
        x = torch.randn(n, heads + 2 * kvh, hd, generator=gen).to(rt)
        return x, x.to(DEV).split([heads, kvh, kvh], 1)

    def append(x, parts, base, pos):
        """base: cache row of position 0"""
        q = torch.empty(len(pos), heads, hd, dtype=rt, device=DEV)
        ops.qk_norm_rope(engine, *parts, gqd, gkd, EPS, td, q, kc, vc, 256, row_base=_i32(base), positions=_i32(pos))
        want, tol = normed_rotated(x[:, :heads], gq, table[pos], EPS, rt == F16)
        check(q, want, tol, "q")
        at = [b + p for b, p in zip(base, pos)]
        want, tol = normed_rotated(x[:, heads:heads + kvh], gk, table[pos], EPS, kt == F16)
        check(kc[at], want, tol, "k")
        return q

    # the shared prompt: rows at positions 0 .. prefix - 1 of cache rows 0 ..
    x, parts = rows(prefix)
    q = append(x, parts, [0] * prefix, list(range(prefix)))
    out = torch.empty_like(q)
    ops.prompt_attention(engine, q, kc, vc, out, 1, prefix)
    want, tol = attend(q.cpu(), kc[:prefix].cpu(), vc[:prefix].cpu(), range(1, prefix + 1), *f16)
    check(out, want, tol, "prompt")
    # each request's own prompt, here as decode steps behind the prefix
    lens = [0, 0]
    for step in range(3):
        x, parts = rows(2)
        # position prefix + len of request s lies in cache row prefix + s cap + len
        q = append(x, parts, [s * cap for s in range(2)], [prefix + n for n in lens])
        lens = [n + 1 for n in lens]
        out = torch.empty_like(q)
        ops.prefix_attention(engine, q, kc, vc, out, 0, prefix, cap, row_base=_i32([prefix + s * cap for s in range(2)]),
                             seq_lens=_i32(lens))
        for s in range(2):
            at = list(range(prefix)) + [prefix + s * cap + i for i in range(lens[s])]
            want, tol = attend(q[s:s + 1].cpu(), kc[at].cpu(), vc[at].cpu(), [len(at)], *f16)
            check(out[s:s + 1], want, tol, (step, s))
    assert U16 > U32 and math.isfinite(float(out.float().sum()))
