"""Sizes at the limits of the packed-row operators, checked on the host."""
import pytest

from janus_amd import _lib
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
