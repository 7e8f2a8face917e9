"""Host checks of the packed-row operators: refused before any device work."""
import ctypes as C

import pytest
import torch

from janus_amd import _lib, ops

F32, F16 = _lib.DT_F32, _lib.DT_F16
P = 0x10000


@pytest.fixture()
def vctx():
    lib = _lib.load()
    h = C.c_void_p()
    assert lib.janus_create(-1, C.byref(h)) == _lib.OK
    yield lib, h
    lib.janus_destroy(h)


PROMPT = dict(q=P, dtype=F16, k=P, v=P, kv=F16, out=P, rows=4, nseq=2, heads=8, kv_heads=2, hd=128, max_seq=64,
              start=P, base=P, lens=P, hint=0, scale=0.0)
PREFIX = dict(q=P, dtype=F16, k=P, v=P, kv=F16, out=P, batch=4, heads=8, kv_heads=2, hd=128, row=0, length=10,
              seq_len=0, max_seq=64, base=P, lens=P, hint=0, scale=0.0)
HEADS = dict(q=P, k=P, v=P, dtype=F32, qs=0, ks=0, vs=0, gq=P, gk=P, eps=1e-5, table=P, out=2 * P, out_dt=F32, kc=P,
             vc=P, kv=F16, rows=4, heads=8, kv_heads=2, hd=128, position=0, max_seq=64, base=P, pos=P)
BOTH = [("janus_prompt_attention", PROMPT), ("janus_prefix_attention", PREFIX)]


def _call(vctx, name, good, **changed):
    lib, ctx = vctx
    assert set(changed) <= set(good)
    status = getattr(lib, name)(ctx, *{**good, **changed}.values())
    return status, lib.janus_last_error(ctx).decode()


@pytest.mark.parametrize("name,good", BOTH + [("janus_qk_norm_rope", HEADS)])
def test_good_calls_reach_the_device_check(vctx, name, good):
    assert _call(vctx, name, good)[0] == _lib.E_NO_DEVICE
    assert getattr(vctx[0], name)(None, *good.values()) == _lib.E_INVALID_ARG


@pytest.mark.parametrize("name,good", BOTH)
def test_attention_refusals(vctx, name, good):
    for buf in ("q", "k", "v", "out"):
        assert _call(vctx, name, good, **{buf: None})[0] == _lib.E_INVALID_ARG
        status, said = _call(vctx, name, good, **{buf: P + 8})
        assert status == _lib.E_INVALID_ARG and "aligned" in said
    for bad in (dict(dtype=_lib.DT_Q8_0), dict(kv=7), dict(dtype=F16, kv=F32)):
        assert _call(vctx, name, good, **bad)[0] == _lib.E_UNSUPPORTED_DTYPE
    for bad in (dict(heads=9), dict(heads=0), dict(kv_heads=0), dict(hd=96), dict(hd=256), dict(heads=1 << 17, kv_heads=1)):
        assert _call(vctx, name, good, **bad)[0] == _lib.E_INVALID_DIM
    for fine in (dict(dtype=F32), dict(dtype=F32, kv=F32), dict(hd=64), dict(base=None), dict(scale=0.3)):
        assert _call(vctx, name, good, **fine)[0] == _lib.E_NO_DEVICE


def test_prompt_rows(vctx):
    for empty in (dict(rows=0), dict(nseq=0)):
        assert _call(vctx, "janus_prompt_attention", PROMPT, **empty)[0] == _lib.OK
    assert _call(vctx, "janus_prompt_attention", PROMPT, start=None, rows=5)[0] == _lib.E_INVALID_DIM
    assert _call(vctx, "janus_prompt_attention", PROMPT, start=None, lens=None, rows=130)[0] == _lib.E_KV_OVERFLOW
    assert _call(vctx, "janus_prompt_attention", PROMPT, start=None, lens=None, rows=128)[0] == _lib.E_NO_DEVICE


def test_prefix_lengths(vctx):
    assert _call(vctx, "janus_prefix_attention", PREFIX, batch=0)[0] == _lib.OK
    assert _call(vctx, "janus_prefix_attention", PREFIX, lens=None, seq_len=65)[0] == _lib.E_KV_OVERFLOW
    assert _call(vctx, "janus_prefix_attention", PREFIX, row=1 << 31)[0] == _lib.E_INVALID_DIM
    assert _call(vctx, "janus_prefix_attention", PREFIX, length=1 << 31)[0] == _lib.E_INVALID_DIM
    far = dict(seq_len=1 << 31, max_seq=0xffffffff)
    assert _call(vctx, "janus_prefix_attention", PREFIX, lens=None, **far)[0] == _lib.E_INVALID_DIM
    assert _call(vctx, "janus_prefix_attention", PREFIX, **far)[0] == _lib.E_NO_DEVICE   # not looked at beside a table


def test_head_refusals(vctx):
    name = "janus_qk_norm_rope"
    for buf in ("q", "k", "v", "table", "out", "kc", "vc"):
        assert _call(vctx, name, HEADS, **{buf: None})[0] == _lib.E_INVALID_ARG
    for bad in (dict(dtype=2), dict(out_dt=8), dict(kv=14)):
        assert _call(vctx, name, HEADS, **bad)[0] == _lib.E_UNSUPPORTED_DTYPE
    for bad in (dict(hd=0), dict(hd=7), dict(hd=1026), dict(heads=0), dict(kv_heads=0), dict(qs=1023), dict(ks=255),
                dict(vs=1), dict(rows=1 << 26)):
        assert _call(vctx, name, HEADS, **bad)[0] == _lib.E_INVALID_DIM
    assert _call(vctx, name, HEADS, pos=None, position=64)[0] == _lib.E_KV_OVERFLOW
    assert _call(vctx, name, HEADS, rows=0)[0] == _lib.OK
    # in place: contiguous rows of one type only
    assert _call(vctx, name, HEADS, out=P)[0] == _lib.E_NO_DEVICE
    assert _call(vctx, name, HEADS, out=P, out_dt=F16)[0] == _lib.E_INVALID_ARG
    assert _call(vctx, name, HEADS, out=P, qs=1536)[0] == _lib.E_INVALID_ARG
    for fine in (dict(gq=None, gk=None), dict(hd=96), dict(hd=1024), dict(qs=1536, ks=1536, vs=1536), dict(kv_heads=3)):
        assert _call(vctx, name, HEADS, **fine)[0] == _lib.E_NO_DEVICE


def test_tensor_checks():
    """The Python wrappers refuse shapes, types and devices that the C call could not see."""
    eng = ops.ComputeEngine(-1)
    eng.device = 0
    q, kv = torch.zeros(4, 8, 64), torch.zeros(32, 2, 64)
    idx = torch.zeros(5, dtype=torch.int32)
    with pytest.raises(ValueError):   # CPU tensors
        ops.prompt_attention(eng, q, kv, kv, q, 1, 32)
    with pytest.raises(ValueError):
        ops.prefix_attention(eng, q, kv, kv, q, 0, 8, 8)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(eng, q, kv[:4], kv[:4], None, None, 1e-5, torch.zeros(8 * 64), q, kv, kv, 8)
    with pytest.raises(ValueError, match="rows, heads, head_dim"):
        ops.prompt_attention(eng, q.view(4, 512), kv, kv, q, 1, 32)
    with pytest.raises(ValueError, match="key and value caches"):
        ops.prompt_attention(eng, q, kv, kv.half(), q, 1, 32)
    with pytest.raises(ValueError, match="q_start"):
        ops._table(idx.long(), torch.int32, 5, 0, "q_start")
    with pytest.raises(ValueError, match="at least 6"):
        ops._table(idx, torch.int32, 6, 0, "q_start")
    eng.device = -1   # that of CPU tensors: sizes are looked at next
    for kw in (dict(nseq=-1, max_seq_len=8), dict(nseq=1, max_seq_len=-1), dict(nseq=5, max_seq_len=8)):
        with pytest.raises(ValueError, match="below 0"):
            ops.prompt_attention(eng, q, kv, kv, q, **kw)
    for kw in (dict(max_seq_len=-1), dict(max_seq_len=8, seq_len=-1), dict(max_seq_len=9, seq_len=1)):
        with pytest.raises(ValueError, match="below 0"):
            ops.prefix_attention(eng, q, kv, kv, q, 0, 8, **kw)
    for row, n in ((-1, 4), (0, 33), (30, 3)):
        with pytest.raises(ValueError, match="beyond the cache"):
            ops.prefix_attention(eng, q, kv, kv, q, row, n, 8)
    for size in (-1, 9):
        with pytest.raises(ValueError, match="below 0"):
            ops.qk_norm_rope(eng, q, kv[:4], kv[:4], None, None, 1e-5, torch.zeros(9 * 64), q, kv, kv, size)
