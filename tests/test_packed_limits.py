"""Sizes at the limits of the packed-row operators, checked on the host."""
import pytest
import torch

from janus_amd import _lib, ops
from test_packed_args import HEADS, PREFIX, PROMPT, _call, vctx  # noqa: F401 (fixture)


@pytest.mark.parametrize("heads,kv_heads,rows,fits", [
    (1, 1, (2 ** 26 - 4) // 3, True), (1, 1, (2 ** 26 - 4) // 3 + 1, False), (2, 1, 2 ** 24 - 1, True),
    (2, 1, 2 ** 24, False), (32, 8, (2 ** 26 - 4) // 48, True), (32, 8, 2 ** 26 // 48 + 1, False)])
@pytest.mark.parametrize("hd", [64, 96])
def test_rows_of_head_norms(vctx, heads, kv_heads, rows, fits, hd):  # noqa: F811
    """One launch holds rows * (heads + 2 kv_heads) <= 2^26 - 4 heads: four to a
    workgroup of 256 lanes, below 2^32 lanes in all."""
    status, said = _call(vctx, "janus_qk_norm_rope", HEADS, heads=heads, kv_heads=kv_heads, rows=rows, hd=hd)
    assert status == (_lib.E_NO_DEVICE if fits else _lib.E_INVALID_DIM)
    assert fits or "more rows" in said


@pytest.mark.parametrize("name,good,rows,seqs", [("janus_prompt_attention", PROMPT, "rows", "nseq"),
                                                 ("janus_prefix_attention", PREFIX, "batch", "batch")])
def test_sizes_of_an_attention(vctx, name, good, rows, seqs):  # noqa: F811
    """rows * heads below 2^25, sequences * kv_heads below 2^24: refused before a device is looked for."""
    for n, fits in ((2 ** 25 // 32 - 1, True), (2 ** 25 // 32, False), (2 ** 32 - 1, False)):
        status, said = _call(vctx, name, good, heads=32, kv_heads=2, **{rows: n})
        assert status == (_lib.E_NO_DEVICE if fits else _lib.E_INVALID_DIM), n
        assert fits or "2^25" in said
    for n, fits in ((2 ** 24 - 1, True), (2 ** 24, False)):
        status, said = _call(vctx, name, good, heads=1, kv_heads=1, **{seqs: n})
        assert status == (_lib.E_NO_DEVICE if fits else _lib.E_INVALID_DIM), n
        assert fits or "2^24" in said
    assert _call(vctx, name, good, **{rows: 0}, **({seqs: 2 ** 25} if seqs != rows else {}))[0] == _lib.OK


def test_numbers_beyond_32_bits():
    """The library takes 32 bits; what does not fit is refused, not cut."""
    eng = ops.ComputeEngine(-1)   # CPU tensors are on its device: every good call reaches the library's device check
    q, kv, far = torch.zeros(4, 8, 64), torch.zeros(32, 2, 64), 2 ** 32 + 8
    i4 = torch.zeros(4, dtype=torch.int32)

    def prompt(nseq=4, max_seq_len=8, base=i4):
        ops.prompt_attention(eng, q, kv, kv, q, nseq, max_seq_len, row_base=base, seq_lens=base)

    def prefix(max_seq_len=8, seq_len=0):
        ops.prefix_attention(eng, q, kv, kv, q, 0, 8, max_seq_len, seq_len=seq_len, row_base=i4)

    def heads(key=kv[:4], value=kv[:4], query=q, position=0):
        ops.qk_norm_rope(eng, query, key, value, None, None, 1e-5, torch.zeros(8 * 64), torch.zeros(4, 8, 64), kv, kv, 8,
                         position=position)

    for call in (prompt, prefix, heads):
        with pytest.raises(ops.JanusError, match="device"):
            call()
    with pytest.raises(ops.JanusError, match="device"):
        prompt(max_seq_len=2 ** 32 - 1)
    # rows 2^32 elements apart, of a meta tensor: only shape, strides and type are looked at
    wide_kv, wide_q = (torch.empty_strided((4, n, 64), (2 ** 32, 64, 1), device="meta") for n in (2, 8))
    for bad in (lambda: prompt(max_seq_len=far), lambda: prompt(nseq=far, max_seq_len=0, base=None),
                lambda: prefix(max_seq_len=far), lambda: prefix(seq_len=far, max_seq_len=2 ** 32 - 1),
                lambda: heads(position=far), lambda: heads(position=-2 ** 32), lambda: heads(key=wide_kv),
                lambda: heads(value=wide_kv), lambda: heads(query=wide_q)):
        with pytest.raises(ValueError, match="32 bits"):
            bad()
