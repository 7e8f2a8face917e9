"""Sizes at the limits of the packed-row operators, checked on the host."""
import pytest

from janus_amd import _lib
from test_packed_args import HEADS, _call, vctx  # noqa: F401 (fixture)


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
