"""Python mirror of janus-engine's operator layer over libjanus_hip.

Names, argument order and error behaviour follow the reference's
`compute::ops` functions (crates/janus-engine/src/compute/ops/mod.rs:31-43)
with the engine/encoder/pipeline-cache arguments folded into one
`ComputeEngine`. Buffers are torch tensors on the GPU (torch provides the
device memory and the stream; all arithmetic runs in the HIP kernels).
Errors raise `JanusError` carrying the reference-equivalent status code.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib
from ._lib import (DT_F16, DT_F32, DT_Q4_0, DT_Q4_K, DT_Q5_K, DT_Q6_K, DT_Q8_0, TIE_LAST,  # noqa: F401
                   TIE_WGSL, WEIGHT_FTZ_F16, JanusError, check)

_TORCH_DT = {torch.float32: DT_F32, torch.float16: DT_F16}


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("janus_amd ops take GPU tensors")
    if not t.is_contiguous():
        raise ValueError("janus_amd ops take contiguous tensors")
    return t.data_ptr()


def _dt(t: torch.Tensor) -> int:
    try:
        return _TORCH_DT[t.dtype]
    except KeyError:
        raise ValueError(f"unsupported activation dtype {t.dtype}") from None


class ComputeEngine:
    """ComputeEngine::new (compute/engine.rs:27-83).

    Owns a janus context on `device`, bound to torch's current stream so
    ordering with torch allocations and copies is implicit. `device=-1`
    creates a validation-only context (host-side argument checks, no GPU).
    """

    def __init__(self, device: int = 0):
        self.lib = _lib.load()
        self.device = device
        h = C.c_void_p()
        check(self.lib.janus_create(device, C.byref(h)))
        self.ctx = h
        if device >= 0:
            self.bind_stream()

    def bind_stream(self, stream: Optional[torch.cuda.Stream] = None) -> None:
        s = stream if stream is not None else torch.cuda.current_stream(self.device)
        check(self.lib.janus_set_stream(self.ctx, C.c_void_p(s.cuda_stream)), self.ctx)

    def sync(self) -> None:
        check(self.lib.janus_sync(self.ctx), self.ctx)

    def workspace_bytes(self) -> tuple[int, int]:
        """(attention, small-M GEMM) workspace sizes of the context."""
        a, g = C.c_size_t(), C.c_size_t()
        check(self.lib.janus_workspace_bytes(self.ctx, C.byref(a), C.byref(g)), self.ctx)
        return a.value, g.value

    def close(self) -> None:
        if self.ctx:
            self.lib.janus_destroy(self.ctx)
            self.ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, status: int) -> None:
        check(status, self.ctx)


class GpuTensor:
    """GpuTensor (compute/tensor.rs:4-7): an uploaded, library-owned weight.

    `data` holds the tensor exactly as a GGUF file stores it (F32/F16 values,
    or Q4_0/Q8_0/Q4_K/Q5_K/Q6_K blocks) for logical shape [n rows][k cols].
    A Q6_K upload reports F16 afterwards, as the reference's loader does.
    """

    def __init__(self, engine: ComputeEngine, ggml_type: int, n: int, k: int, data, flags: int = 0):
        self.engine = engine
        self.ggml_type = ggml_type
        self.n, self.k = n, k
        buf = np.ascontiguousarray(data).view(np.uint8).reshape(-1)
        h = C.c_void_p()
        engine._check(engine.lib.janus_weight_upload(engine.ctx, ggml_type, n, k, buf.ctypes.data,
                                                     buf.nbytes, flags, C.byref(h)))
        self.handle = h
        # Q6_K is stored as binary16 after upload (compute/engine.rs:800-831)
        t = C.c_int()
        engine._check(engine.lib.janus_weight_info(h, C.byref(t), None, None, None))
        self.ggml_type = t.value

    def dequant(self) -> torch.Tensor:
        out = torch.empty(self.n, self.k, dtype=torch.float32, device=f"cuda:{self.engine.device}")
        self.engine._check(self.engine.lib.janus_weight_dequant(self.engine.ctx, self.handle, _ptr(out)))
        return out

    def free(self) -> None:
        if self.handle:
            self.engine.lib.janus_weight_free(self.engine.ctx, self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


# ---- matrix products (ops/quantized.rs:63-186) -----------------------------

def gemm_auto(engine: ComputeEngine, matrix_a: torch.Tensor, matrix_b: GpuTensor, output: torch.Tensor,
              batch_size: int, m: int, k: int, n: int) -> None:
    engine._check(engine.lib.janus_gemm_auto(engine.ctx, _ptr(matrix_a), _dt(matrix_a), matrix_b.handle,
                                             _ptr(output), _dt(output), batch_size, m, k, n))


def gemm_residual(engine: ComputeEngine, a: torch.Tensor, w: GpuTensor, residual: torch.Tensor,
                  output: torch.Tensor, rows: int) -> None:
    engine._check(engine.lib.janus_gemm_residual(engine.ctx, _ptr(a), _dt(a), w.handle, _ptr(residual),
                                                 _ptr(output), rows, w.k, w.n))


# ---- activations / elementwise (ops/activation.rs, ops/elementwise.rs) -------

def rmsnorm(engine, input, output, weights, batch_size: int, hidden_dim: int, epsilon: float) -> None:
    engine._check(engine.lib.janus_rmsnorm(engine.ctx, _ptr(input), _ptr(output), _dt(output), _ptr(weights),
                                           batch_size, hidden_dim, epsilon))


def silu(engine, input, output, size: int) -> None:
    engine._check(engine.lib.janus_silu(engine.ctx, _ptr(input), _ptr(output), size))


def elementwise_mul(engine, tensor_a, tensor_b, output, size: int) -> None:
    engine._check(engine.lib.janus_elementwise_mul(engine.ctx, _ptr(tensor_a), _ptr(tensor_b), _ptr(output), size))


def add_tensors(engine, tensor_a, tensor_b, output, size: int) -> None:
    engine._check(engine.lib.janus_add_tensors(engine.ctx, _ptr(tensor_a), _ptr(tensor_b), _ptr(output), size))


def swiglu(engine, gate, up, output, size: int) -> None:
    engine._check(engine.lib.janus_swiglu(engine.ctx, _ptr(gate), _ptr(up), _ptr(output), _dt(output), size))


# ---- RoPE (ops/rope.rs:48-115) -----------------------------------------------

def create_rope_cache(engine, max_seq_len: int, head_dim: int, theta_base: float) -> torch.Tensor:
    """Model::create_rope_cache (model/transformer/constructor.rs:454-489)."""
    t = torch.empty(max_seq_len * head_dim, dtype=torch.float32, device=f"cuda:{engine.device}")
    engine._check(engine.lib.janus_rope_table(engine.ctx, _ptr(t), max_seq_len, head_dim, theta_base))
    return t


def rope(engine, input, output, rope_cache, batch_size: int, num_heads: int, head_dim: int, position: int,
         positions: Optional[torch.Tensor] = None) -> None:
    engine._check(engine.lib.janus_rope(engine.ctx, _ptr(input), _ptr(output), _ptr(rope_cache), batch_size,
                                        num_heads, head_dim, position, _ptr(positions)))


# ---- KV cache (compute/cache/core.rs) -------------------------------------------

class KVCache:
    """KVCache::new / update / buffers (compute/cache/core.rs:60-324).

    Layout per cache: [num_layers][batch_size * max_seq_len][num_kv_heads][head_dim];
    sequence b owns rows [b * max_seq_len, (b + 1) * max_seq_len) of each layer.
    """

    def __init__(self, engine, batch_size: int, num_layers: int, max_seq_len: int, num_kv_heads: int,
                 head_dim: int, dtype: torch.dtype = torch.float32):
        self.engine = engine
        self.batch_size, self.num_layers, self.max_seq_len = batch_size, num_layers, max_seq_len
        self.num_kv_heads, self.head_dim = num_kv_heads, head_dim
        self.dtype = dtype
        shape = (num_layers, batch_size * max_seq_len, num_kv_heads, head_dim)
        dev = f"cuda:{engine.device}"
        self.key_cache = torch.zeros(shape, dtype=dtype, device=dev)
        self.value_cache = torch.zeros(shape, dtype=dtype, device=dev)
        self.position = 0

    def update(self, new_key, new_value, layer_idx: int, position: int) -> None:
        engine = self.engine
        engine._check(engine.lib.janus_kv_update(
            engine.ctx, _ptr(new_key), _ptr(new_value), _ptr(self.key_cache[layer_idx]),
            _ptr(self.value_cache[layer_idx]), _dt(self.key_cache), self.batch_size, self.num_kv_heads,
            self.head_dim, position, self.max_seq_len, None, None))
        self.position = position + 1

    def current_position(self) -> int:
        return self.position

    def buffers(self):
        return self.key_cache, self.value_cache

    def reset(self) -> None:
        self.position = 0


def kv_update(engine, k_new, v_new, k_cache, v_cache, batch: int, kv_heads: int, head_dim: int, position: int,
              max_seq_len: int, row_base=None, positions=None) -> None:
    engine._check(engine.lib.janus_kv_update(engine.ctx, _ptr(k_new), _ptr(v_new), _ptr(k_cache), _ptr(v_cache),
                                             _dt(k_cache), batch, kv_heads, head_dim, position, max_seq_len,
                                             _ptr(row_base), _ptr(positions)))


# ---- attention (ops/attention.rs:78-235) ------------------------------------------

def compute_attention(engine, query, key_cache, value_cache, output, batch_size: int, seq_len: int,
                      max_seq_len: int, num_heads: int, num_kv_heads: int, head_dim: int,
                      row_base: Optional[torch.Tensor] = None, seq_lens: Optional[torch.Tensor] = None,
                      max_len_hint: int = 0, scale: float = 0.0) -> None:
    """One decode query per sequence against one layer's cache slice."""
    engine._check(engine.lib.janus_attention(
        engine.ctx, _ptr(query), _ptr(key_cache), _ptr(value_cache), _dt(key_cache), _ptr(output), batch_size,
        num_heads, num_kv_heads, head_dim, seq_len, max_seq_len, _ptr(row_base), _ptr(seq_lens), max_len_hint,
        scale))


def compute_attention_noalloc(engine, query, key_cache, value_cache, output, batch_size: int, seq_len: int,
                              max_seq_len: int, num_heads: int, num_kv_heads: int, head_dim: int,
                              row_base: Optional[torch.Tensor] = None, seq_lens: Optional[torch.Tensor] = None,
                              max_len_hint: int = 0, scale: float = 0.0) -> None:
    """compute_attention through the allocation-free entry point (fixed
    per-device scratch; janus_attention_noalloc in include/janus_hip.h)."""
    engine._check(engine.lib.janus_attention_noalloc(
        engine.ctx, _ptr(query), _ptr(key_cache), _ptr(value_cache), _dt(key_cache), _ptr(output), batch_size,
        num_heads, num_kv_heads, head_dim, seq_len, max_seq_len, _ptr(row_base), _ptr(seq_lens), max_len_hint,
        scale))


# ---- heads and attention of packed rows ----------------------------------------------

_U32 = 0xffffffff   # the library's sizes


def _buf(t: torch.Tensor, dev: int, name: str) -> int:
    """Address of a contiguous tensor on the engine's device."""
    if t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous tensor on cuda:{dev} expected, got {t.device}, strides {t.stride()}")
    return t.data_ptr()


def _table(t: Optional[torch.Tensor], dtype: torch.dtype, least: int, dev: int, name: str) -> Optional[int]:
    """Address of a table of at least `least` values, or None."""
    if t is None:
        return None
    if t.dtype is not dtype or t.numel() < least:
        raise ValueError(f"{name}: at least {least} values of {dtype} expected, got {t.numel()} of {t.dtype}")
    if t.get_device() != dev or not t.is_contiguous():
        return _buf(t, dev, name)
    return t.data_ptr()


def _stride(t: torch.Tensor, rows: int, heads: int, hd: int, dev: int, name: str) -> int:
    """Elements from a row to the next of [rows, heads, head_dim] whose heads lie
    one behind the other, such as a part of a fused product's rows."""
    row, head, one = t.stride()
    if t.get_device() != dev or (one != 1 and hd != 1) or (head != hd and heads != 1) or (row < heads * hd and rows > 1):
        raise ValueError(f"{name}: [rows, heads, head_dim] on cuda:{dev} with contiguous rows expected, got {t.device}, "
                         f"strides {t.stride()}")
    if row > _U32 and rows > 1:
        raise ValueError(f"{name}: rows {row} elements apart, beyond 32 bits")
    return row if rows > 1 else heads * hd


def _caches(key_cache: torch.Tensor, value_cache: torch.Tensor, hd: int, dev: int) -> tuple[int, int, int, int, int]:
    """(K address, V address, dtype, rows, kv heads) of one layer's caches [rows, kv_heads, head_dim]."""
    shape, dtype = key_cache.shape, key_cache.dtype
    if len(shape) != 3 or shape[2] != hd or value_cache.shape != shape or value_cache.dtype is not dtype:
        raise ValueError(f"key and value caches: [rows, kv_heads, {hd}] of one type expected, got {tuple(shape)} and "
                         f"{tuple(value_cache.shape)}")
    return (_buf(key_cache, dev, "key_cache"), _buf(value_cache, dev, "value_cache"),
            _TORCH_DT[dtype] if dtype in _TORCH_DT else _dt(key_cache), shape[0], shape[1])


def _three(t: torch.Tensor, name: str):
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{name}: [rows, heads, head_dim] expected, got {tuple(shape)}")
    return shape


def qk_norm_rope(engine, query, key, value, q_gamma, k_gamma, epsilon: float, rope_cache, output, key_cache,
                 value_cache, max_seq_len: int, position: int = 0, row_base: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None) -> None:
    """RMS norm of each query and key head (q_gamma, k_gamma: [head_dim], or None
    for no norm), rotation, and the append of K and V to the cache, in one pass
    (janus_qk_norm_rope in include/janus_hip.h). query, key and value are [rows,
    heads, head_dim], also as parts of one fused product's rows; output [rows,
    heads, head_dim] receives the rotated queries and may be query. K and V of row
    r go to cache row row_base[r] + position; a negative row_base[r] is padding and
    appends nothing."""
    dev = engine.device
    shape = _three(query, "query")
    rows, heads, hd = shape
    kc, vc, kv_dt, cache_rows, kvh = _caches(key_cache, value_cache, hd, dev)
    kv_shape, dtype = (rows, kvh, hd), query.dtype
    if key.shape != kv_shape or value.shape != kv_shape or output.shape != shape:
        raise ValueError(f"key and value: {kv_shape}, output: {tuple(shape)} expected, got {tuple(key.shape)}, "
                         f"{tuple(value.shape)}, {tuple(output.shape)}")
    if key.dtype is not dtype or value.dtype is not dtype:
        raise ValueError("query, key and value: one type expected")
    if max_seq_len < 0 or (row_base is None and rows * max_seq_len > cache_rows):
        raise ValueError("max_seq_len below 0, or without row_base fewer cache rows than max_seq_len for each row")
    if max_seq_len > _U32 or (positions is None and not -0x80000000 <= position <= _U32):
        raise ValueError("max_seq_len or position beyond 32 bits")
    f32, i32 = torch.float32, torch.int32
    status = engine.lib.janus_qk_norm_rope(
        engine.ctx, query.data_ptr(), key.data_ptr(), value.data_ptr(), _dt(query),
        _stride(query, rows, heads, hd, dev, "query"), _stride(key, rows, kvh, hd, dev, "key"),
        _stride(value, rows, kvh, hd, dev, "value"), _table(q_gamma, f32, hd, dev, "q_gamma"),
        _table(k_gamma, f32, hd, dev, "k_gamma"), epsilon, _table(rope_cache, f32, max_seq_len * hd, dev, "rope_cache"),
        _buf(output, dev, "output"), _dt(output), kc, vc, kv_dt, rows, heads, kvh, hd, position, max_seq_len,
        _table(row_base, i32, rows, dev, "row_base"), _table(positions, i32, rows, dev, "positions"))
    if status:
        engine._check(status)


def prompt_attention(engine, query, key_cache, value_cache, output, nseq: int, max_seq_len: int,
                     q_start: Optional[torch.Tensor] = None, row_base: Optional[torch.Tensor] = None,
                     seq_lens: Optional[torch.Tensor] = None, max_len_hint: int = 0, scale: float = 0.0) -> None:
    """Causal attention of the packed rows of nseq sequences against one layer's
    cache (janus_prompt_attention in include/janus_hip.h): sequence s has the
    rows [q_start[s], q_start[s + 1]) of query [rows, heads, head_dim], the last
    of its seq_lens[s] positions, which lie in the cache from row_base[s] on."""
    dev = engine.device
    shape = _three(query, "query")
    rows, heads, hd = shape
    kc, vc, kv_dt, cache_rows, kvh = _caches(key_cache, value_cache, hd, dev)
    if output.shape != shape or output.dtype is not query.dtype:
        raise ValueError("output: the query's shape and type expected")
    if nseq < 0 or max_seq_len < 0 or (row_base is None and nseq * max_seq_len > cache_rows):
        raise ValueError("nseq or max_seq_len below 0, or without row_base fewer cache rows than max_seq_len for each "
                         "sequence")
    if max_seq_len > _U32 or nseq > _U32:
        raise ValueError("nseq or max_seq_len beyond 32 bits")
    i32 = torch.int32
    status = engine.lib.janus_prompt_attention(
        engine.ctx, _buf(query, dev, "query"), _dt(query), kc, vc, kv_dt, _buf(output, dev, "output"), rows, nseq,
        heads, kvh, hd, max_seq_len, _table(q_start, i32, nseq + 1, dev, "q_start"),
        _table(row_base, i32, nseq, dev, "row_base"), _table(seq_lens, i32, nseq, dev, "seq_lens"), max_len_hint,
        scale)
    if status:
        engine._check(status)


def prefix_attention(engine, query, key_cache, value_cache, output, prefix_row: int, prefix_len: int,
                     max_seq_len: int, seq_len: int = 0, row_base: Optional[torch.Tensor] = None,
                     seq_lens: Optional[torch.Tensor] = None, max_len_hint: int = 0, scale: float = 0.0) -> None:
    """One decode query per sequence against a prefix that all of them share,
    cache rows [prefix_row, prefix_row + prefix_len), and its own positions behind
    it, [row_base[b], row_base[b] + seq_lens[b]) (janus_prefix_attention in
    include/janus_hip.h)."""
    dev = engine.device
    shape = _three(query, "query")
    batch, heads, hd = shape
    kc, vc, kv_dt, cache_rows, kvh = _caches(key_cache, value_cache, hd, dev)
    if output.shape != shape or output.dtype is not query.dtype:
        raise ValueError("output: the query's shape and type expected")
    if prefix_row < 0 or prefix_len < 0 or prefix_row + prefix_len > cache_rows:
        raise ValueError("the prefix lies beyond the cache")
    if max_seq_len < 0 or seq_len < 0 or (row_base is None and (seq_lens is not None or seq_len)
                                          and batch * max_seq_len > cache_rows):
        raise ValueError("max_seq_len or seq_len below 0, or without row_base fewer cache rows than max_seq_len for each "
                         "sequence")
    if max_seq_len > _U32 or (seq_lens is None and seq_len > _U32):
        raise ValueError("max_seq_len or seq_len beyond 32 bits")
    i32 = torch.int32
    status = engine.lib.janus_prefix_attention(
        engine.ctx, _buf(query, dev, "query"), _dt(query), kc, vc, kv_dt, _buf(output, dev, "output"), batch, heads,
        kvh, hd, prefix_row, prefix_len, seq_len, max_seq_len, _table(row_base, i32, batch, dev, "row_base"),
        _table(seq_lens, i32, batch, dev, "seq_lens"), max_len_hint, scale)
    if status:
        engine._check(status)


# ---- a cache of 4-bit values -----------------------------------------------------------

def _fp4_caches(k_cache, k_scales, v_cache, v_scales, hd, dev: int):
    """(addresses of K, its scales, V, its scales, rows, kv heads) of one layer's 4-bit
    caches: values [rows, kv_heads, head_dim / 2] and scales [rows, kv_heads, head_dim / 32]."""
    shape, u8 = k_cache.shape, torch.uint8
    if len(shape) != 3 or shape[2] * 2 != hd or v_cache.shape != shape:
        raise ValueError(f"4-bit caches: [rows, kv_heads, {hd} / 2] expected, got {tuple(shape)} and "
                         f"{tuple(v_cache.shape)}")
    scales = (shape[0], shape[1], hd // 32)
    if k_scales.shape != scales or v_scales.shape != scales:
        raise ValueError(f"scales: {scales} expected, got {tuple(k_scales.shape)} and {tuple(v_scales.shape)}")
    if k_cache.dtype is not u8 or k_scales.dtype is not u8 or v_cache.dtype is not u8 or v_scales.dtype is not u8:
        raise ValueError("4-bit caches and scales: torch.uint8 expected")
    return (_buf(k_cache, dev, "k_cache"), _buf(k_scales, dev, "k_scales"), _buf(v_cache, dev, "v_cache"),
            _buf(v_scales, dev, "v_scales"), shape[0], shape[1])


def kv_update_fp4(engine, key, value, k_cache, k_scales, v_cache, v_scales, max_seq_len: int, position: int = 0,
                  row_base: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None) -> None:
    """Append rows of K and V to a cache of 4-bit values (janus_kv_update_fp4 in
    include/janus_hip.h). key and value are [rows, kv_heads, head_dim] of float32 or
    float16, also as parts of one fused product's rows; row r goes to cache row
    row_base[r] + positions[r] (without row_base r * max_seq_len, without positions
    `position`). The caches are torch.uint8: values [cache rows, kv_heads, head_dim / 2],
    scales [cache rows, kv_heads, head_dim / 32]; a cache of zeros holds zeros."""
    dev = engine.device
    shape = _three(key, "key")
    rows, kvh, hd = shape
    kc, ks, vc, vs, cache_rows, cache_heads = _fp4_caches(k_cache, k_scales, v_cache, v_scales, hd, dev)
    if value.shape != shape or value.dtype is not key.dtype or cache_heads != kvh:
        raise ValueError(f"value: {tuple(shape)} of key's type and caches of {kvh} heads expected, got "
                         f"{tuple(value.shape)} and {cache_heads}")
    if max_seq_len < 0 or (row_base is None and rows * max_seq_len > cache_rows):
        raise ValueError("max_seq_len below 0, or without row_base fewer cache rows than max_seq_len for each row")
    if max_seq_len > _U32 or (positions is None and not 0 <= position <= _U32):
        raise ValueError("max_seq_len or position beyond 32 bits")
    i32 = torch.int32
    status = engine.lib.janus_kv_update_fp4(
        engine.ctx, key.data_ptr(), value.data_ptr(), _dt(key), _stride(key, rows, kvh, hd, dev, "key"),
        _stride(value, rows, kvh, hd, dev, "value"), kc, ks, vc, vs, rows, kvh, hd, cache_rows, position, max_seq_len,
        _table(row_base, i32, rows, dev, "row_base"), _table(positions, i32, rows, dev, "positions"))
    if status:
        engine._check(status)


def kv_read_fp4(engine, k_cache, k_scales, v_cache, v_scales, k_out, v_out, first_row: int = 0,
                rows: Optional[torch.Tensor] = None) -> None:
    """Rows of a 4-bit cache as float32 or float16 values, which hold them exactly
    (janus_kv_read_fp4 in include/janus_hip.h): k_out and v_out [n, kv_heads, head_dim]
    receive cache row rows[r], or first_row + r."""
    dev = engine.device
    shape = _three(k_out, "k_out")
    n, kvh, hd = shape
    kc, ks, vc, vs, cache_rows, cache_heads = _fp4_caches(k_cache, k_scales, v_cache, v_scales, hd, dev)
    if v_out.shape != shape or v_out.dtype is not k_out.dtype or cache_heads != kvh:
        raise ValueError(f"v_out: {tuple(shape)} of k_out's type and caches of {kvh} heads expected, got "
                         f"{tuple(v_out.shape)} and {cache_heads}")
    if rows is None and not 0 <= first_row <= cache_rows - n:
        raise ValueError("the rows lie beyond the cache")
    status = engine.lib.janus_kv_read_fp4(engine.ctx, kc, ks, vc, vs, _buf(k_out, dev, "k_out"),
                                          _buf(v_out, dev, "v_out"), _dt(k_out), n, kvh, hd, cache_rows,
                                          first_row if rows is None else 0, _table(rows, torch.int32, n, dev, "rows"))
    if status:
        engine._check(status)


def fp4_attention(engine, query, k_cache, k_scales, v_cache, v_scales, output, nseq: int, max_seq_len: int,
                  q_start: Optional[torch.Tensor] = None, row_base: Optional[torch.Tensor] = None,
                  seq_lens: Optional[torch.Tensor] = None, max_len_hint: int = 0, scale: float = 0.0) -> None:
    """prompt_attention over a 4-bit cache (janus_fp4_attention in include/janus_hip.h):
    causal attention of the packed rows of nseq sequences, sequence s with the rows
    [q_start[s], q_start[s + 1]) of query [rows, heads, head_dim] (rows / nseq each
    without q_start: a decode step has one), the last of its seq_lens[s] positions,
    which lie in the cache from row_base[s] on."""
    dev = engine.device
    shape = _three(query, "query")
    rows, heads, hd = shape
    kc, ks, vc, vs, cache_rows, kvh = _fp4_caches(k_cache, k_scales, v_cache, v_scales, hd, dev)
    if output.shape != shape or output.dtype is not query.dtype:
        raise ValueError("output: the query's shape and type expected")
    if nseq < 0 or max_seq_len < 0 or (row_base is None and nseq * max_seq_len > cache_rows):
        raise ValueError("nseq or max_seq_len below 0, or without row_base fewer cache rows than max_seq_len for each "
                         "sequence")
    if max_seq_len > _U32 or nseq > _U32 or not 0 <= max_len_hint <= _U32:
        raise ValueError("nseq, max_seq_len or max_len_hint beyond 32 bits")
    i32 = torch.int32
    status = engine.lib.janus_fp4_attention(
        engine.ctx, _buf(query, dev, "query"), _dt(query), kc, ks, vc, vs, _buf(output, dev, "output"), rows, nseq,
        heads, kvh, hd, cache_rows, max_seq_len, _table(q_start, i32, nseq + 1, dev, "q_start"),
        _table(row_base, i32, nseq, dev, "row_base"), _table(seq_lens, i32, nseq, dev, "seq_lens"), max_len_hint,
        scale)
    if status:
        engine._check(status)


# ---- beam search -------------------------------------------------------------------------

def beam_select(engine, logits, scores: Optional[torch.Tensor], out_scores, out_parents, out_tokens) -> None:
    """The best continuations of each request's beams (janus_beam_select in
    include/janus_hip.h). logits [batch * beams, vocab] float32 (or [batch, beams,
    vocab]), scores [batch, beams] float32 or None for zeros; out_scores (float32), out_parents and
    out_tokens (int32), [batch, n], receive the n largest of scores + log_softmax(logits)
    of each request in descending order, equal ones by beam, then token. A beam whose score
    is -infinity has ended. out_scores may be scores where n is beams."""
    dev = engine.device
    if out_scores.dim() != 2 or (scores is not None and (scores.dim() != 2 or out_scores.shape[0] != scores.shape[0])):
        raise ValueError(f"scores: [batch, beams] and out_scores: [batch, n] expected, got "
                         f"{'none' if scores is None else tuple(scores.shape)} and {tuple(out_scores.shape)}")
    batch, n = out_scores.shape
    vocab = logits.shape[-1] if logits.dim() else 0
    beams = scores.shape[1] if scores is not None else logits.numel() // (batch * vocab) if batch * vocab else 1
    if logits.numel() != batch * beams * vocab:
        raise ValueError(f"logits: {batch} x {beams} rows expected, got {tuple(logits.shape)}")
    if out_parents.shape != out_scores.shape or out_tokens.shape != out_scores.shape:
        raise ValueError("out_parents and out_tokens: out_scores' shape expected")
    f32, i32 = torch.float32, torch.int32
    if logits.dtype is not f32 or (scores is not None and scores.dtype is not f32) or out_scores.dtype is not f32 or out_parents.dtype is not i32 \
            or out_tokens.dtype is not i32:
        raise ValueError("logits and scores: torch.float32, parents and tokens: torch.int32 expected")
    status = engine.lib.janus_beam_select(engine.ctx, _buf(logits, dev, "logits"),
                                          None if scores is None else _buf(scores, dev, "scores"),
                                          _buf(out_scores, dev, "out_scores"), _buf(out_parents, dev, "out_parents"),
                                          _buf(out_tokens, dev, "out_tokens"), batch, beams, vocab, n)
    if status:
        engine._check(status)


def kv_reorder(engine, caches: Sequence[torch.Tensor], beams: int, max_seq_len: int, row_base: torch.Tensor,
               parents: torch.Tensor, seq_lens: Optional[torch.Tensor] = None, layers: int = 0) -> None:
    """Every beam goes on from its parent, in place (janus_kv_reorder in
    include/janus_hip.h): slot i of a request, the cache rows from row_base[i] on, takes
    the first seq_lens[i] (max_seq_len) rows that the request's slot parents[i] held.
    caches: up to 8 tensors of one number of rows, [rows, ...] or, with `layers`, [layers,
    rows, ...] (K and V, a 4-bit cache's scales beside them). row_base, parents and
    seq_lens hold `beams` values for each request, those of a request one behind the
    other; parents count within the request."""
    dev, lead = engine.device, 1 if layers else 0
    if not caches or len(caches) > 8:
        raise ValueError(f"1 to 8 caches expected, got {len(caches)}")
    slots = parents.numel()
    if beams < 1 or layers < 0 or max_seq_len < 0 or slots % beams:
        raise ValueError("beams below 1, layers or max_seq_len below 0, or parents not of whole requests")
    if max_seq_len > _U32 or layers > _U32:
        raise ValueError("max_seq_len or layers beyond 32 bits")
    rows = caches[0].shape[lead] if caches[0].dim() > lead else 0
    sizes = []
    for c in caches:
        shape = c.shape
        if len(shape) <= lead or shape[lead] != rows or (lead and shape[0] != layers):
            raise ValueError(f"caches: {f'[{layers}, {rows}, ...]' if lead else f'[{rows}, ...]'} expected, got {tuple(shape)}")
        sizes.append(c.numel() * c.element_size() // max(1, rows * (layers or 1)))
    if not rows:
        return
    k = len(caches)
    bufs = (C.c_void_p * k)(*[_buf(c, dev, "cache") for c in caches])
    i32 = torch.int32
    status = engine.lib.janus_kv_reorder(
        engine.ctx, k, bufs, (C.c_uint64 * k)(*sizes), layers or 1, slots // beams, beams, rows, max_seq_len,
        _table(row_base, i32, slots, dev, "row_base"), _table(parents, i32, slots, dev, "parents"),
        _table(seq_lens, i32, slots, dev, "seq_lens"))
    if status:
        engine._check(status)


# ---- embedding and sampling ---------------------------------------------------------

def embed_tokens(engine, table: GpuTensor, token_ids: Sequence[int], output) -> None:
    """Model::embed_tokens (model/transformer/embedding.rs:16-198)."""
    ids = np.ascontiguousarray(np.asarray(token_ids, dtype=np.uint32))
    engine._check(engine.lib.janus_embed(engine.ctx, table.handle, ids.ctypes.data, len(ids), _ptr(output)))


def argmax(engine, logits, output, vocab_size: int, batch_size: int, tie_rule: int = TIE_WGSL) -> None:
    """ops::argmax (ops/argmax.rs:50-107); tie_rule TIE_LAST gives Sampler::argmax."""
    engine._check(engine.lib.janus_argmax(engine.ctx, _ptr(logits), _ptr(output), vocab_size, batch_size, tie_rule))


def repetition_penalty(engine, logits, vocab_size: int, context: torch.Tensor, penalty: float) -> None:
    engine._check(engine.lib.janus_repetition_penalty(engine.ctx, _ptr(logits), vocab_size, _ptr(context),
                                                      context.numel(), penalty))
