"""Host checks of the 4-bit cache's operators and of beam search: refused before any device work."""
import ctypes as C

import pytest
import torch

from janus_amd import _lib, ops
from fp4_ref import decode, encode
from test_packed_args import vctx  # noqa: F401 (fixture)

F32, F16 = _lib.DT_F32, _lib.DT_F16
P, FAR = 0x10000, 1 << 44
CACHE = dict(kc=P, ks=P, vc=P, vs=P)
STORE = dict(k=P, v=P, dtype=F32, k_stride=0, v_stride=0, **CACHE, rows=4, kv_heads=2, hd=128, cache_rows=256, position=0,
             max_seq=64, base=P, pos=P)
READ = dict(**CACHE, ko=P, vo=P, dtype=F16, rows=4, kv_heads=2, hd=128, cache_rows=256, first=0, table=P)
ATTEND = dict(q=P, dtype=F16, **CACHE, out=P, rows=4, nseq=2, heads=8, kv_heads=2, hd=128, cache_rows=256, max_seq=64,
              start=P, base=P, lens=P, hint=0, scale=0.0)
SELECT = dict(logits=P, scores=P, out=P, parents=P, tokens=P, batch=2, beams=4, vocab=1000, n=8)
FP4 = [("janus_kv_update_fp4", STORE), ("janus_kv_read_fp4", READ), ("janus_fp4_attention", ATTEND)]


def _call(vctx, name, good, **changed):  # noqa: F811
    lib, ctx = vctx
    assert set(changed) <= set(good)
    status = getattr(lib, name)(ctx, *{**good, **changed}.values())
    return status, lib.janus_last_error(ctx).decode()


def _reorder(vctx, buffers=(P, FAR), row_bytes=(256, 32), layers=2, groups=3, beams=4, cache_rows=100, max_seq=8, base=P,  # noqa: F811
             parents=P, lens=P, **other):
    lib, ctx = vctx
    k = len(buffers)
    args = dict(n=k, buffers=(C.c_void_p * k)(*buffers), row_bytes=(C.c_uint64 * k)(*row_bytes), **other)
    status = lib.janus_kv_reorder(ctx, args["n"], args["buffers"], args["row_bytes"], layers, groups, beams, cache_rows,
                                  max_seq, base, parents, lens)
    return status, lib.janus_last_error(ctx).decode()


@pytest.mark.parametrize("name,good", FP4 + [("janus_beam_select", SELECT)])
def test_good_calls_reach_the_device_check(vctx, name, good):  # noqa: F811
    assert _call(vctx, name, good)[0] == _lib.E_NO_DEVICE
    assert getattr(vctx[0], name)(None, *good.values()) == _lib.E_INVALID_ARG


@pytest.mark.parametrize("name,good", FP4)
def test_cache_refusals(vctx, name, good):  # noqa: F811
    for buf in CACHE:
        assert _call(vctx, name, good, **{buf: None})[0] == _lib.E_INVALID_ARG
        status, said = _call(vctx, name, good, **{buf: P + (2 if buf[1] == "s" else 8)})
        assert status == _lib.E_INVALID_ARG and "aligned" in said
    assert _call(vctx, name, good, ks=P + 4, vs=P + 12)[0] == _lib.E_NO_DEVICE
    for bad in (dict(hd=0), dict(hd=80), dict(hd=1056), dict(kv_heads=0), dict(kv_heads=65537), dict(cache_rows=2 ** 31 + 1)):
        assert _call(vctx, name, good, **bad)[0] == _lib.E_INVALID_DIM, bad
    assert _call(vctx, name, good, dtype=_lib.DT_Q4_0)[0] == _lib.E_UNSUPPORTED_DTYPE


def test_store_refusals(vctx):  # noqa: F811
    name = "janus_kv_update_fp4"
    for bad in (dict(k=None), dict(v=None), dict(k=P + 2), dict(v=P + 1, dtype=F16)):
        assert _call(vctx, name, STORE, **bad)[0] == _lib.E_INVALID_ARG, bad
    for bad in (dict(k_stride=255), dict(v_stride=1), dict(rows=2 ** 24)):
        assert _call(vctx, name, STORE, **bad)[0] == _lib.E_INVALID_DIM, bad
    assert _call(vctx, name, STORE, pos=None, position=64)[0] == _lib.E_KV_OVERFLOW
    for fine in (dict(rows=0), dict(cache_rows=0)):
        assert _call(vctx, name, STORE, **fine)[0] == _lib.OK
    for fine in (dict(k=P + 2, v=P + 2, dtype=F16), dict(hd=32), dict(hd=1024), dict(k_stride=1000, v_stride=300),
                 dict(rows=2 ** 24 - 1), dict(base=None, pos=None, position=63)):
        assert _call(vctx, name, STORE, **fine)[0] == _lib.E_NO_DEVICE, fine


def test_read_refusals(vctx):  # noqa: F811
    name = "janus_kv_read_fp4"
    for bad in (dict(ko=None), dict(vo=None), dict(ko=P + 8), dict(vo=P + 4)):
        assert _call(vctx, name, READ, **bad)[0] == _lib.E_INVALID_ARG, bad
    for bad in (dict(table=None, first=253), dict(table=None, first=2 ** 32 - 1)):
        assert _call(vctx, name, READ, **bad)[0] == _lib.E_KV_OVERFLOW
    assert _call(vctx, name, READ, table=None, first=252)[0] == _lib.E_NO_DEVICE
    assert _call(vctx, name, READ, rows=2 ** 24)[0] == _lib.E_INVALID_DIM
    assert _call(vctx, name, READ, rows=0)[0] == _lib.OK


def test_attention_refusals(vctx):  # noqa: F811
    name = "janus_fp4_attention"
    for bad in (dict(q=None), dict(out=None), dict(q=P + 8), dict(out=P + 4)):
        assert _call(vctx, name, ATTEND, **bad)[0] == _lib.E_INVALID_ARG, bad
    for bad in (dict(heads=9), dict(heads=0), dict(hd=32), dict(hd=96), dict(hd=256), dict(heads=1 << 17, kv_heads=1),
                dict(start=None, rows=5), dict(rows=2 ** 22), dict(nseq=2 ** 21, rows=8)):
        assert _call(vctx, name, ATTEND, **bad)[0] == _lib.E_INVALID_DIM, bad
    assert _call(vctx, name, ATTEND, start=None, lens=None, rows=130)[0] == _lib.E_KV_OVERFLOW
    for fine in (dict(rows=0), dict(nseq=0)):
        assert _call(vctx, name, ATTEND, **fine)[0] == _lib.OK
    for fine in (dict(nseq=2 ** 21 - 1), dict(rows=2 ** 22 - 1), dict(dtype=F32), dict(hd=64), dict(base=None), dict(scale=0.3), dict(start=None, lens=None, rows=128)):
        assert _call(vctx, name, ATTEND, **fine)[0] == _lib.E_NO_DEVICE, fine


def test_select_refusals(vctx):  # noqa: F811
    name = "janus_beam_select"
    for buf in ("logits", "out", "parents", "tokens"):
        assert _call(vctx, name, SELECT, **{buf: None})[0] == _lib.E_INVALID_ARG
    for bad in (dict(beams=0), dict(beams=65), dict(vocab=0), dict(vocab=2 ** 29), dict(n=0), dict(n=65),
                dict(beams=1, vocab=7, n=8), dict(batch=2 ** 24)):
        assert _call(vctx, name, SELECT, **bad)[0] == _lib.E_INVALID_DIM, bad
    assert _call(vctx, name, SELECT, batch=0)[0] == _lib.OK
    for fine in (dict(scores=None), dict(beams=64, n=64), dict(beams=2, vocab=4), dict(vocab=2 ** 29 - 1, batch=1)):
        assert _call(vctx, name, SELECT, **fine)[0] == _lib.E_NO_DEVICE, fine


def test_select_takes_as_many_requests_as_one_launch(vctx):  # noqa: F811
    # 512 lanes for each request and for each part of a row, fewer than 2^32 in all
    small = dict(beams=1, vocab=7, n=1)
    assert _call(vctx, "janus_beam_select", SELECT, batch=2 ** 23, **small)[0] == _lib.E_INVALID_DIM
    assert _call(vctx, "janus_beam_select", SELECT, batch=2 ** 23 - 1, **small)[0] == _lib.E_NO_DEVICE


def test_reorder_refusals(vctx):  # noqa: F811
    assert _reorder(vctx)[0] == _lib.E_NO_DEVICE
    for bad in (dict(buffers=(P, None)), dict(base=None), dict(parents=None)):
        assert _reorder(vctx, **bad)[0] == _lib.E_INVALID_ARG, bad
    nine = dict(buffers=(P,) * 9, row_bytes=(1,) * 9)
    for bad in (nine, dict(row_bytes=(0, 1)), dict(row_bytes=(1, 2 ** 30 + 1)), dict(beams=0), dict(beams=33),
                dict(cache_rows=2 ** 31 + 1), dict(layers=2 ** 23), dict(groups=2 ** 22), dict(groups=2 ** 30, layers=1)):
        assert _reorder(vctx, **bad)[0] == _lib.E_INVALID_DIM, bad
    for fine in (dict(buffers=(), row_bytes=()), dict(layers=0), dict(groups=0), dict(cache_rows=0), dict(max_seq=0),
                 dict(beams=1)):
        assert _reorder(vctx, **fine)[0] == _lib.OK, fine
    for fine in (dict(lens=None), dict(row_bytes=(1, 2 ** 30)), dict(beams=32)):
        assert _reorder(vctx, **fine)[0] == _lib.E_NO_DEVICE, fine
    size = 2 * 100 * 256   # of the first buffer: the second may begin behind it, or end before it
    for other in (P + size, P - 2 * 100 * 32):
        assert _reorder(vctx, (P, other))[0] == _lib.E_NO_DEVICE
    for other in (P, P + 1, P + size - 1, P - 2 * 100 * 32 + 1):
        status, said = _reorder(vctx, (P, other))
        assert status == _lib.E_INVALID_ARG and "overlap" in said, other


@pytest.fixture()
def cpu_engine():
    return ops.ComputeEngine(-1)   # CPU tensors are on its device: good calls reach the library's device check


def _caches(rows=32, kvh=2, hd=64):
    return [torch.zeros(rows, kvh, hd // d, dtype=torch.uint8) for d in (2, 32, 2, 32)]


def test_fp4_tensor_checks(cpu_engine):
    eng, i4 = cpu_engine, torch.zeros(4, dtype=torch.int32)
    kv, q, far = torch.zeros(4, 2, 64), torch.zeros(4, 8, 64), 2 ** 32

    def store(caches=None, key=kv, value=kv, max_seq_len=8, **kw):
        ops.kv_update_fp4(eng, key, value, *(caches or _caches()), max_seq_len, **kw)

    def read(caches=None, k_out=kv, v_out=kv, **kw):
        ops.kv_read_fp4(eng, *(caches or _caches()), k_out, v_out, **kw)

    def attend(caches=None, query=q, output=q, nseq=4, max_seq_len=8, **kw):
        ops.fp4_attention(eng, query, *(caches or _caches()), output, nseq, max_seq_len, **kw)

    for call in (store, read, attend):
        with pytest.raises(ops.JanusError, match="device"):
            call()
        a, s, b, t = _caches()
        for bad in ([a[:, :, :31], s, b, t], [a, s[:31], b, t], [a, s, b[:31], t], [a, s, b, t[:, :1]], [a.char(), s, b, t],
                    [a, s.float(), b, t], [a.transpose(0, 1).contiguous().transpose(0, 1), s, b, t], _caches(kvh=3)[:2] + [b, t]):
            with pytest.raises(ValueError):
                call(bad)
    for bad in (dict(key=kv.view(4, 128)), dict(value=kv.half()), dict(value=kv[:3]), dict(caches=_caches(kvh=1)),
                dict(max_seq_len=-1), dict(max_seq_len=9), dict(max_seq_len=far, row_base=i4), dict(position=-1),
                dict(position=far), dict(row_base=i4[:3]), dict(row_base=i4.long()), dict(positions=i4.float()),
                dict(key=kv.expand(4, 2, 64).transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            store(**bad)
    for bad in (dict(v_out=kv.half()), dict(v_out=kv[:3]), dict(first_row=-1), dict(first_row=29), dict(rows=i4[:3])):
        with pytest.raises(ValueError):
            read(**bad)
    for bad in (dict(output=q[:3]), dict(output=q.half()), dict(nseq=-1), dict(nseq=5), dict(max_seq_len=-1), dict(max_seq_len=9),
                dict(max_seq_len=far, row_base=i4), dict(nseq=far, max_seq_len=0), dict(q_start=i4), dict(seq_lens=i4[:2]),
                dict(max_len_hint=-1), dict(max_len_hint=far)):
        with pytest.raises(ValueError):
            attend(**bad)


def test_beam_tensor_checks(cpu_engine):
    eng = cpu_engine
    logits, scores = torch.zeros(6, 50), torch.zeros(2, 3)
    out, idx = torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int32)

    def select(logits=logits, scores=scores, out=out, parents=idx, tokens=idx):
        ops.beam_select(eng, logits, scores, out, parents, tokens)

    for call in (select, lambda: select(logits.view(2, 3, 50))):
        with pytest.raises(ops.JanusError, match="device"):
            call()
    for bad in (dict(scores=scores.view(6)), dict(out=out[:1]), dict(logits=logits[:5]), dict(parents=idx[:, :3]),
                dict(tokens=idx[:1]), dict(logits=logits.half()), dict(scores=scores.double()), dict(parents=idx.long()),
                dict(logits=torch.zeros(50, 6).T)):
        with pytest.raises(ValueError):
            select(**bad)

    k = torch.zeros(40, 2, 64, dtype=torch.float16)
    i6 = torch.arange(6, dtype=torch.int32)

    def reorder(caches=(k, k.clone()), beams=3, max_seq_len=5, row_base=i6, parents=i6, **kw):
        ops.kv_reorder(eng, list(caches), beams, max_seq_len, row_base, parents, **kw)

    for call in (reorder, lambda: reorder((k.view(4, 10, 2, 64), k.clone().view(4, 10, 2, 64)), layers=4), lambda: reorder((k, k[:, 0, 0].contiguous()))):
        with pytest.raises(ops.JanusError, match="device"):
            call()
    reorder((k[:0],))
    with pytest.raises(ops.JanusError, match="overlap"):
        reorder((k, k))
    for bad in (dict(caches=()), dict(caches=(k,) * 9), dict(caches=(k, k[:39])), dict(beams=0), dict(beams=4), dict(max_seq_len=-1),
                dict(max_seq_len=2 ** 32), dict(layers=-1), dict(layers=3), dict(row_base=i6[:5]), dict(parents=i6.long()),
                dict(seq_lens=i6[:4]), dict(caches=(k.transpose(1, 2),))):
        with pytest.raises(ValueError):
            reorder(**bad)


def test_the_reference_of_the_format():
    """Codes of known values: ties go to the even code, the scale follows the largest."""
    x = torch.zeros(1, 32)
    x[0, :10] = torch.tensor([4, 0.25, 0.75, -1.25, 1.75, 2.5, 3.5, 5, -6, 0.3])
    codes, scales = encode(x)
    assert scales.tolist() == [[127]]
    assert decode(codes, scales)[0, :10].tolist() == [4, 0, 1, -1, 2, 2, 4, 4, -6, 0.5]
    for top, byte, value in ((7.0, 127, 6.0), (7.01, 128, 8.0), (1e9, 140, 6 * 2.0 ** 13), (1e-12, 104, 0.0)):
        x[:] = 0
        x[0, 3] = -top
        codes, scales = encode(x)
        assert scales.item() == byte and decode(codes, scales)[0, 3].item() == -value
    for odd in (float("nan"), float("inf"), -float("inf")):
        x[0, 3] = odd
        codes, scales = encode(x)
        assert scales.item() == 255 and not codes.any() and decode(codes, scales).isnan().all()
    codes = torch.tensor([[0x21] * 16], dtype=torch.uint8)
    for byte, pair in ((104, [0.5 * 2.0 ** -23, 2.0 ** -23]), (103, [0.0, 2.0 ** -24]), (102, [0.0, 0.0]), (0, [0.0, 0.0]), (140, [4096.0, 8192.0])):
        assert decode(codes, torch.tensor([[byte]], dtype=torch.uint8))[0, :2].tolist() == pair
