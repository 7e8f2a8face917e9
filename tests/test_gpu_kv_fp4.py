"""janus_kv_update_fp4 and janus_kv_read_fp4: every byte and value against the format's definition."""
import math

import pytest
import torch

from janus_amd import ops
from fp4_ref import decode, encode, random_cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _caches(rows, kvh, hd, fill=0):
    return [torch.full((rows, kvh, hd // d), fill, dtype=torch.uint8, device=DEV) for d in (2, 32, 2, 32)]


def _rows(gen, rows, kvh, hd, dtype):
    """Values over many binades, values next to and at the borders between codes, zeros."""
    x = torch.randn(rows, kvh, hd, generator=gen) * 2.0 ** torch.randint(-10, 8, (rows, kvh, hd // 32, 1), generator=gen).expand(
        -1, -1, -1, 32).reshape(rows, kvh, hd)
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 4, 0.0, -0.0])
    pick = border[torch.randint(0, len(border), x.shape, generator=gen)] * torch.randn(x.shape, generator=gen).sign()
    x = torch.where(torch.rand(x.shape, generator=gen) < 0.3, pick, x)
    x[..., ::31] = torch.nextafter(x[..., ::31], torch.tensor(math.inf))
    x[0, 0, :32] = 0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("kvh,hd", [(8, 128), (2, 64), (1, 32), (3, 96), (1, 1024), (32, 128)])
@pytest.mark.parametrize("rows", [1, 37])
def test_append_and_read_back(engine, dtype, kvh, hd, rows):
    gen = torch.Generator().manual_seed(rows + hd)
    k, v = (_rows(gen, rows, kvh, hd, dtype) for _ in range(2))
    caches = _caches(2 * rows + 3, kvh, hd, 77)
    base = torch.randperm(rows, generator=gen) * 2
    pos = torch.randint(0, 2, (rows,), generator=gen)
    ops.kv_update_fp4(engine, k.to(DEV), v.to(DEV), *caches, 2, row_base=_i32(base.tolist()), positions=_i32(pos.tolist()))
    want = [torch.full(c.shape, 77, dtype=torch.uint8) for c in caches]
    at = base + pos
    want[0][at], want[1][at] = encode(k)
    want[2][at], want[3][at] = encode(v)
    for got, w in zip(caches, want):
        assert torch.equal(got.cpu(), w)
    for out_dtype in (torch.float16, torch.float32):
        ko, vo = (torch.empty(rows, kvh, hd, dtype=out_dtype, device=DEV) for _ in range(2))
        ops.kv_read_fp4(engine, *caches, ko, vo, rows=_i32(at.tolist()))
        assert torch.equal(ko.cpu().double(), decode(want[0][at], want[1][at]))
        assert torch.equal(vo.cpu().double(), decode(want[2][at], want[3][at]))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_ranges(engine, dtype):
    """Blocks from the smallest to beyond the largest scale, and ones with an infinity or NaN."""
    gen = torch.Generator().manual_seed(3)
    tops = [2.0 ** e for e in range(-26, 16)] + ([1e-38, 1e-45, 1e20, 3e38, 57344.0, 57345.0, 65535.0] if dtype == torch.float32 else [65504.0])
    tops += [math.inf, -math.inf, math.nan, 0.0]
    x = torch.randn(len(tops), 1, 32, generator=gen).clamp(-1, 1)
    x = torch.where(torch.tensor(tops).isfinite()[:, None, None], x * torch.tensor(tops).nan_to_num(0, 0, 0)[:, None, None], x)
    x[:, 0, 5] = torch.tensor(tops)
    x = x.to(dtype)
    caches = _caches(len(tops), 1, 32, 9)
    ops.kv_update_fp4(engine, x.to(DEV), -x.to(DEV), *caches, 1)
    for i, sign in ((0, 1), (2, -1)):
        codes, scales = encode(sign * x)
        assert torch.equal(caches[i + 1].cpu(), scales)
        # a float32 value below the smallest normal one may count as zero of either sign
        assert torch.equal(decode(caches[i].cpu(), scales).nan_to_num(1e9), decode(codes, scales).nan_to_num(1e9))


def test_parts_of_a_fused_product(engine):
    gen = torch.Generator().manual_seed(4)
    for dtype, pad in ((torch.float16, 0), (torch.float16, 5), (torch.float32, 0), (torch.float32, 3)):
        rows, heads, kvh, hd = 9, 4, 2, 64
        qkv = torch.randn(rows, (heads + 2 * kvh) * hd + pad, generator=gen).to(dtype)   # odd strides: values one by one
        dev = qkv.to(DEV)
        k, v = (dev[:, i * hd:(i + kvh) * hd].unflatten(1, (kvh, hd)) for i in (heads, heads + kvh))
        caches = _caches(rows * 4, kvh, hd)
        ops.kv_update_fp4(engine, k, v, *caches, 4, position=2)
        codes, scales = encode(v.cpu())
        assert torch.equal(caches[2][2::4].cpu(), codes) and torch.equal(caches[3][2::4].cpu(), scales)
        codes, scales = encode(k.cpu())
        assert torch.equal(caches[0][2::4].cpu(), codes) and torch.equal(caches[1][2::4].cpu(), scales)
        assert not caches[0][0::4].any() and not caches[3][3::4].any()


def test_rows_that_are_left_out(engine):
    """Padding, positions outside the slot and rows beyond the cache write nothing."""
    kvh, hd = 2, 64
    x = torch.ones(8, kvh, hd, device=DEV)
    caches = _caches(20, kvh, hd, 7)
    base, pos = [-1, 0, 4, 8, 16, 16, 2 ** 31 - 1, -2 ** 31], [0, 4, -1, 1, 3, 2 ** 31 - 1, 3, 2]
    ops.kv_update_fp4(engine, x, x, *caches, 4, row_base=_i32(base), positions=_i32(pos))
    written = {9, 19}
    for c in caches:
        for r in range(20):
            assert (c[r] != 7).any() == (r in written), r
    caches = _caches(6, kvh, hd, 7)   # the cache ends inside a slot
    ops.kv_update_fp4(engine, x[:2], x[:2], *caches, 4, row_base=_i32([3, 4]), positions=_i32([2, 2]))
    assert (caches[0][5] != 7).any() and (caches[0][:5] == 7).all()
    out = torch.full((4, kvh, hd), 5.0, device=DEV)
    ops.kv_read_fp4(engine, *caches, out, out.clone(), rows=_i32([-1, 5, 6, 2 ** 31 - 1]))
    assert (out[[0, 2, 3]] == 5).all() and (out[1] == 1).all()


def test_read_of_foreign_scales(engine):
    """Scale bytes that no append writes: below 104 the values are rounded to binary16, above 140 the block is NaN."""
    gen = torch.Generator().manual_seed(6)
    kc, _ = random_cache(gen, 256, 1, 32)
    ks = torch.arange(256, dtype=torch.uint8).view(256, 1, 1)
    for dtype in (torch.float16, torch.float32):
        ko, vo = (torch.empty(250, 1, 32, dtype=dtype, device=DEV) for _ in range(2))
        ops.kv_read_fp4(engine, kc.to(DEV), ks.to(DEV), kc.flip(0).to(DEV), ks.flip(0).to(DEV), ko, vo, first_row=6)
        for got, c, s in ((ko, kc, ks), (vo, kc.flip(0), ks.flip(0))):
            want = decode(c, s)[6:]
            assert torch.equal(got.cpu().double().nan_to_num(1e9), want.nan_to_num(1e9))
            assert torch.equal(got.cpu().isnan(), want.isnan())


def test_offsets_beyond_32_bits(engine):
    """Cache rows whose values lie beyond 2^32 bytes."""
    kvh, hd = 32, 128
    rows = 2 ** 32 // (kvh * hd // 2) + 5
    kc, vc = (torch.zeros(rows, kvh, hd // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(rows, kvh, hd // 32, dtype=torch.uint8, device=DEV) for _ in range(2))
    x = torch.randn(1, kvh, hd, generator=torch.Generator().manual_seed(7))
    ops.kv_update_fp4(engine, x.to(DEV), -x.to(DEV), kc, ks, vc, vs, 8, row_base=_i32([rows - 4]), positions=_i32([3]))
    ko, vo = (torch.empty(1, kvh, hd, device=DEV) for _ in range(2))
    ops.kv_read_fp4(engine, kc, ks, vc, vs, ko, vo, first_row=rows - 1)
    want = decode(*encode(x))
    assert torch.equal(ko.cpu().double(), want) and torch.equal(vo.cpu().double(), -want)
    assert not kc[:8].any() and not vs[:8].any()


def test_captured_append_and_read(engine):
    """A captured append and read, replayed with other rows, positions and slots, equal the eager calls."""
    gen = torch.Generator().manual_seed(8)
    kvh, hd, n = 4, 64, 6
    k, v = (torch.randn(n, kvh, hd, generator=gen).half().to(DEV) for _ in range(2))
    base, pos, at = _i32([0] * n), _i32([0] * n), _i32([0] * n)
    caches, ko, vo = _caches(40, kvh, hd), *(torch.zeros(n, kvh, hd, device=DEV) for _ in range(2))

    def step():
        ops.kv_update_fp4(engine, k, v, *caches, 5, row_base=base, positions=pos)
        ops.kv_read_fp4(engine, *caches, ko, vo, rows=at)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        engine.bind_stream(stream)
        try:
            step()
            stream.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                step()
            for i in range(4):
                k.copy_(torch.randn(n, kvh, hd, generator=gen).half())
                v.copy_(torch.randn(n, kvh, hd, generator=gen).half())
                slot, p = torch.randperm(8, generator=gen)[:n] * 5, torch.randint(0, 5, (n,), generator=gen)
                base.copy_(_i32(slot.tolist()))
                pos.copy_(_i32(p.tolist()))
                at.copy_(_i32((slot + p).tolist()))
                for c in caches:
                    c.fill_(7)
                g.replay()
                stream.synchronize()
                for got, x, c in ((ko, k, 0), (vo, v, 2)):
                    codes, scales = encode(x.cpu())
                    assert torch.equal(caches[c].cpu()[slot + p], codes) and torch.equal(caches[c + 1].cpu()[slot + p], scales), i
                    assert torch.equal(got.cpu().double(), decode(codes, scales)), i
                    assert (caches[c].cpu() == 7).all(-1).all(-1).sum() >= 40 - n
        finally:
            engine.bind_stream(torch.cuda.default_stream())
