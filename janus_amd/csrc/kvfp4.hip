// kvfp4.hip -- K and V rows into a cache of 4-bit values, and back.
//
// A block of 32 values x of a head has one scale 2^e (byte e + 127):
//   e = floor(log2 max|x|) - 2, one more where max|x| > 1.75 2^floor(log2 max|x|),
//   within [-23, 13],
// and each value goes to the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} 2^e, ties to
// the even code, larger ones to 6 2^e. Scales are powers of two, so nothing is
// rounded before that step and the result is the same whoever computes it. The
// e2m1 values and power-of-two scales are those of the matrix unit's own 4-bit
// format (the Open Compute microscaling formats, whose conversion is floor - 2
// alone; the exception for the top eighth of a binade lowers the relative rms error
// of normal values from 0.115 to 0.112, of uniform ones from 0.144 to 0.099). The
// range of e makes every value a binary16 number, subnormal ones among them.
//
// Pure traffic: a lane holds 8 values, four lanes a block. 8192 rows of 8 heads of 128 dims in
// binary16 are written and read back in 19 us (4.5 TB/s, what a large copy reaches), 32 rows in 14,
// which is two launches.
#include "internal.h"

namespace janus {
namespace {

struct StoreArgs {
    const void *k, *v;
    uint32_t k_stride, v_stride;   // elements from a row to the next
    uint8_t *kc, *ks, *vc, *vs;
    const int32_t *row_base, *positions;
    uint32_t kv_heads, hd, cache_rows, position, max_seq;
    uint32_t blocks;               // workgroups per row
};

template <typename T, bool VEC> __device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
    if constexpr (VEC) {
        typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
        for (int i = 0; i < 8; i += 16 / (int)sizeof(T)) {
            const vec w = *(const vec *)(p + i);
#pragma unroll
            for (int j = 0; j < 16 / (int)sizeof(T); ++j) x[i + j] = (float)w[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)p[i];
    }
}

template <typename T, bool VEC> __global__ __launch_bounds__(256) void kv_store_fp4_kernel(StoreArgs a) {
    const uint32_t row = blockIdx.x / a.blocks;
    const int32_t p = a.positions ? a.positions[row] : (int32_t)a.position;
    const int64_t base = a.row_base ? (int64_t)a.row_base[row] : (int64_t)row * a.max_seq;
    const int64_t at_row = base + p;
    if (p < 0 || (uint32_t)p >= a.max_seq || base < 0 || at_row >= (int64_t)a.cache_rows) return;
    const uint32_t elems = a.kv_heads * a.hd;   // of K, and of V
    uint32_t i = ((blockIdx.x % a.blocks) * blockDim.x + threadIdx.x) * 8u;
    if (i >= 2u * elems) return;                // whole blocks of 32: four lanes leave together
    const bool is_v = i >= elems;
    if (is_v) i -= elems;
    const T *src = is_v ? (const T *)a.v + (size_t)row * a.v_stride : (const T *)a.k + (size_t)row * a.k_stride;
    float x[8];
    load8<T, VEC>(src + i, x);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xb1, 0xf, 0xf, false));   // quad_perm [1,0,3,2]
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4e, 0xf, 0xf, false));   // quad_perm [2,3,0,1]
    const bool odd = top >= 0x7f800000u;        // an infinity or NaN: the block has no values
    const int e = max(-23, min(13, (int)(top >> 23) - 129 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0)));
    const float scale = __uint_as_float((uint32_t)(e + 127) << 23);
    uint32_t code = 0;
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[0], x[1], scale, 0);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[2], x[3], scale, 1);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[4], x[5], scale, 2);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[6], x[7], scale, 3);
    const size_t to = (size_t)at_row * elems + i;
    *(uint32_t *)((is_v ? a.vc : a.kc) + to / 2) = odd ? 0u : code;
    if ((threadIdx.x & 3u) == 0) (is_v ? a.vs : a.ks)[to / 32] = odd ? 255 : (uint8_t)(e + 127);
}

struct ReadArgs {
    const uint8_t *kc, *ks, *vc, *vs;
    void *k, *v;                   // [rows][kv_heads][hd]
    const int32_t *rows;           // cache row of each, or null: first + r
    uint32_t first, cache_rows, elems;
    uint32_t blocks;               // workgroups per row
};

template <typename T> __global__ __launch_bounds__(256) void kv_read_fp4_kernel(ReadArgs a) {
    const uint32_t r = blockIdx.x / a.blocks;
    const int64_t row = a.rows ? (int64_t)a.rows[r] : (int64_t)a.first + r;
    if (row < 0 || row >= (int64_t)a.cache_rows) return;
    uint32_t i = ((blockIdx.x % a.blocks) * blockDim.x + threadIdx.x) * 8u;
    if (i >= 2u * a.elems) return;
    const bool is_v = i >= a.elems;
    if (is_v) i -= a.elems;
    const size_t at = (size_t)row * a.elems + i;
    const uint32_t code = *(const uint32_t *)((is_v ? a.vc : a.kc) + at / 2);
    const uint32_t b = (is_v ? a.vs : a.ks)[at / 32];
    T *out = (T *)(is_v ? a.v : a.k) + (size_t)r * a.elems + i;
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
    // binary16 holds every value that the append wrote; what others wrote is rounded to it
    const bool odd = b > 140u;
    const float s = __uint_as_float(min(b, 140u) << 23);
    const jh2 x[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, s, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, s, 1),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, s, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, s, 3)};
#pragma unroll
    for (int j = 0; j < 8; j += 16 / (int)sizeof(T)) {
        vec w;
#pragma unroll
        for (int t = 0; t < 16 / (int)sizeof(T); ++t) w[t] = odd ? (T)__uint_as_float(0x7fc00000u) : (T)x[(j + t) >> 1][t & 1];
        *(vec *)(out + j) = w;
    }
}

// Lanes of a workgroup, and workgroups per row, for n lanes of a row.
void shape_of(uint32_t lanes, uint32_t *threads, uint32_t *blocks) {
    *threads = lanes >= 256 ? 256 : (lanes + 63) / 64 * 64;
    *blocks = (lanes + *threads - 1) / *threads;
}

}  // namespace

int kv_update_fp4_launch(janus_ctx *ctx, const void *k, const void *v, int in_dt, uint32_t k_stride, uint32_t v_stride,
                         uint8_t *kc, uint8_t *ks, uint8_t *vc, uint8_t *vs, uint32_t rows, uint32_t kv_heads,
                         uint32_t hd, uint32_t cache_rows, uint32_t position, uint32_t max_seq,
                         const int32_t *row_base, const int32_t *positions) {
    StoreArgs a{k, v, k_stride, v_stride, kc, ks, vc, vs, row_base, positions, kv_heads, hd, cache_rows, position,
                max_seq, 1};
    uint32_t threads;
    shape_of(2 * kv_heads * (hd / 8), &threads, &a.blocks);
    const dim3 grid(rows * a.blocks), block(threads);
    const bool vec = (((uintptr_t)k | (uintptr_t)v | (uintptr_t)(k_stride * act_bytes(in_dt)) |
                       (uintptr_t)(v_stride * act_bytes(in_dt))) & 15u) == 0;
    if (in_dt == JANUS_DT_F16) {
        if (vec) hipLaunchKernelGGL((kv_store_fp4_kernel<_Float16, true>), grid, block, 0, ctx->stream, a);
        else hipLaunchKernelGGL((kv_store_fp4_kernel<_Float16, false>), grid, block, 0, ctx->stream, a);
    } else {
        if (vec) hipLaunchKernelGGL((kv_store_fp4_kernel<float, true>), grid, block, 0, ctx->stream, a);
        else hipLaunchKernelGGL((kv_store_fp4_kernel<float, false>), grid, block, 0, ctx->stream, a);
    }
    JANUS_LAUNCH_CHECK(ctx);
    return JANUS_OK;
}

int kv_read_fp4_launch(janus_ctx *ctx, const uint8_t *kc, const uint8_t *ks, const uint8_t *vc, const uint8_t *vs,
                       void *k_out, void *v_out, int out_dt, uint32_t rows, uint32_t kv_heads, uint32_t hd,
                       uint32_t cache_rows, uint32_t first_row, const int32_t *d_rows) {
    ReadArgs a{kc, ks, vc, vs, k_out, v_out, d_rows, first_row, cache_rows, kv_heads * hd, 1};
    uint32_t threads;
    shape_of(2 * kv_heads * (hd / 8), &threads, &a.blocks);
    const dim3 grid(rows * a.blocks), block(threads);
    if (out_dt == JANUS_DT_F16) hipLaunchKernelGGL((kv_read_fp4_kernel<_Float16>), grid, block, 0, ctx->stream, a);
    else hipLaunchKernelGGL((kv_read_fp4_kernel<float>), grid, block, 0, ctx->stream, a);
    JANUS_LAUNCH_CHECK(ctx);
    return JANUS_OK;
}

}  // namespace janus
