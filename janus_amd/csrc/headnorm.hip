// headnorm.hip -- RMS norm of the query and key heads, rotation and KV append
// in one pass.
//
// Row r at position p, head vector x of D values, gain g (or none):
//   y = x / sqrt(mean(x^2) + eps) * g             (y = x without a gain)
//   z_i = y_i c_i - y_{i + D/2} s_i,  z_{i + D/2} = y_i s_i + y_{i + D/2} c_i
// with (c_i, s_i) = table[p][i]. Query heads go to q_out, key heads and the
// untouched value heads to the row's cache row.
//
// Bound by HBM: every value is read and written once. A head is held by the lanes
// that load it, 16 bytes of either half each, so the norm is a sum over 4 to 32
// lanes and the turn stays in a lane. Outputs are stored past the caches: 8192
// binary16 rows of a 32/8/128 product (202 MB) take 37 us (5.4 TB/s; a copy reaches
// 4.7), 40 with ordinary stores; binary32 rows into a binary16 cache (370 MB) 64 and
// 68; 4096 binary16 rows at 32/8/256 (203 MB) 37 and 40. Four heads of a row per lane
// group (the table read once for them) were slower. Head dims and alignments that the
// vectors do not fit take a wavefront per head and a value per load, at a quarter of
// the rate: 8192 binary16 rows at 32/8/96 (152 MB) 160 us, the 202 MB above at odd
// addresses 170; 48 rows of a decode step are bound by the call, 9 us, either way.
#include "internal.h"

namespace janus {
namespace {

struct HeadArgs {
    const void *q, *k, *v;
    uint32_t q_stride, k_stride, v_stride;   // elements from a row to the next
    const float *q_gamma, *k_gamma;
    const float *table;                      // [max_seq][D / 2] (cos, sin)
    void *q_out, *kc, *vc;
    const int32_t *row_base, *positions;
    uint32_t rows, heads, kv_heads, hd, position, max_seq;
    float eps;
};

struct Place {
    uint32_t pos;
    bool rotates, appends;
    size_t cache_row;
};

__device__ __forceinline__ Place place_of(const HeadArgs &a, uint32_t row) {
    const int32_t p = a.positions ? a.positions[row] : (int32_t)a.position;
    const int64_t base = a.row_base ? (int64_t)a.row_base[row] : (int64_t)row * a.max_seq;
    Place r;
    r.rotates = p >= 0 && (uint32_t)p < a.max_seq;
    r.appends = r.rotates && base >= 0;
    r.pos = r.rotates ? (uint32_t)p : 0u;
    r.cache_row = r.appends ? (size_t)base + r.pos : 0;
    return r;
}

// E consecutive values as floats, and back; the address is a multiple of their size (at most 16 bytes).
template <typename T, int E> __device__ __forceinline__ void load_e(const T *p, float (&x)[E]) {
    typedef T vec __attribute__((ext_vector_type(E < 16 / (int)sizeof(T) ? E : 16 / (int)sizeof(T))));
    constexpr int N = sizeof(vec) / sizeof(T);
#pragma unroll
    for (int i = 0; i < E; i += N) {
        const vec v = *(const vec *)(p + i);
#pragma unroll
        for (int j = 0; j < N; ++j) x[i + j] = (float)v[j];
    }
}
template <typename T, int E> __device__ __forceinline__ void store_e(T *p, const float (&x)[E]) {
    typedef T vec __attribute__((ext_vector_type(E < 16 / (int)sizeof(T) ? E : 16 / (int)sizeof(T))));
    constexpr int N = sizeof(vec) / sizeof(T);
#pragma unroll
    for (int i = 0; i < E; i += N) {
        vec v;
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = (T)x[i + j];
        __builtin_nontemporal_store(v, (vec *)(p + i));
    }
}

// D / 2 / E lanes share a head: each holds E values of the first half and the
// E values that they turn with.
template <typename IN, typename OUT, typename KV, int D, int E>
__global__ __launch_bounds__(256) void head_kernel(HeadArgs a) {
    constexpr uint32_t L = D / 2 / E;
    const uint32_t units = a.heads + 2 * a.kv_heads;
    const uint32_t unit = (uint32_t)(((uint64_t)blockIdx.x * 256u + threadIdx.x) / L), at = threadIdx.x % L * E;
    const uint32_t row = unit / units, h = unit % units;
    if (row >= a.rows) return;
    const bool is_q = h < a.heads, is_k = !is_q && h < a.heads + a.kv_heads;
    const uint32_t kh = h - a.heads - (is_k ? 0u : a.kv_heads);
    const IN *src = is_q   ? (const IN *)a.q + (size_t)row * a.q_stride + (size_t)h * D
                    : is_k ? (const IN *)a.k + (size_t)row * a.k_stride + (size_t)kh * D
                           : (const IN *)a.v + (size_t)row * a.v_stride + (size_t)kh * D;
    float x0[E], x1[E];
    load_e<IN, E>(src + at, x0);
    load_e<IN, E>(src + D / 2 + at, x1);
    const Place pl = place_of(a, row);
    const float *gamma = is_q ? a.q_gamma : is_k ? a.k_gamma : nullptr;
    if (gamma) {
        float g0[E], g1[E], s = 0.0f;
        load_e<float, E>(gamma + at, g0);
        load_e<float, E>(gamma + D / 2 + at, g1);
#pragma unroll
        for (int i = 0; i < E; ++i) s = fmaf(x0[i], x0[i], fmaf(x1[i], x1[i], s));
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) s += shfl_xor(s, o);
        const float r = 1.0f / sqrtf(s * (1.0f / D) + a.eps);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            x0[i] = x0[i] * r * g0[i];
            x1[i] = x1[i] * r * g1[i];
        }
    }
    if (is_q || is_k) {
        float cs[2 * E];
        load_e<float, 2 * E>(a.table + ((size_t)pl.pos * (D / 2) + at) * 2, cs);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float p = x0[i], n = x1[i], c = cs[2 * i], s = cs[2 * i + 1];
            x0[i] = p * c - n * s;
            x1[i] = p * s + n * c;
        }
    }
    if (is_q) {
        OUT *o = (OUT *)a.q_out + ((size_t)row * a.heads + h) * D + at;
        if (pl.rotates) {
            store_e<OUT, E>(o, x0);
            store_e<OUT, E>(o + D / 2, x1);
        }
    } else if (pl.appends) {
        KV *o = (KV *)(is_k ? a.kc : a.vc) + (pl.cache_row * a.kv_heads + kh) * D + at;
        store_e<KV, E>(o, x0);
        store_e<KV, E>(o + D / 2, x1);
    }
}

// Any even head dim up to 1024 and any alignment: a wavefront per head.
template <typename IN, typename OUT, typename KV>
__global__ __launch_bounds__(256) void head_any_kernel(HeadArgs a) {
    const uint32_t units = a.heads + 2 * a.kv_heads, half = a.hd / 2, lane = threadIdx.x & 63u;
    const uint64_t unit = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6);
    const uint32_t row = (uint32_t)(unit / units), h = (uint32_t)(unit % units);
    if (row >= a.rows) return;
    const Place pl = place_of(a, row);
    const bool is_q = h < a.heads, is_k = !is_q && h < a.heads + a.kv_heads;
    const uint32_t kh = h - a.heads - (is_k ? 0u : a.kv_heads);
    const IN *src = is_q   ? (const IN *)a.q + (size_t)row * a.q_stride + (size_t)h * a.hd
                    : is_k ? (const IN *)a.k + (size_t)row * a.k_stride + (size_t)kh * a.hd
                           : (const IN *)a.v + (size_t)row * a.v_stride + (size_t)kh * a.hd;
    float x0[8], x1[8], s = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t i = lane + 64u * j;
        x0[j] = i < half ? (float)src[i] : 0.0f;
        x1[j] = i < half ? (float)src[i + half] : 0.0f;
        s = fmaf(x0[j], x0[j], fmaf(x1[j], x1[j], s));
    }
    const float *gamma = is_q ? a.q_gamma : is_k ? a.k_gamma : nullptr;
    const float r = gamma ? 1.0f / sqrtf(wave_sum(s) / (float)a.hd + a.eps) : 1.0f;
    if (is_q ? !pl.rotates : !pl.appends) return;
    const size_t to = is_q ? ((size_t)row * a.heads + h) * a.hd : (pl.cache_row * a.kv_heads + kh) * a.hd;
    KV *kv = (KV *)(is_k ? a.kc : a.vc);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t i = lane + 64u * j;
        if (i >= half) break;
        float p = x0[j], n = x1[j];
        if (gamma) {
            p = p * r * gamma[i];
            n = n * r * gamma[i + half];
        }
        if (is_q || is_k) {
            const float *t = a.table + ((size_t)pl.pos * half + i) * 2;
            const float c = t[0], sn = t[1], y = p * c - n * sn;
            n = p * sn + n * c;
            p = y;
        }
        if (is_q) {
            ((OUT *)a.q_out)[to + i] = (OUT)p;
            ((OUT *)a.q_out)[to + half + i] = (OUT)n;
        } else {
            kv[to + i] = (KV)p;
            kv[to + half + i] = (KV)n;
        }
    }
}

template <typename IN, typename OUT, typename KV, int D>
void launch_dim(janus_ctx *ctx, const HeadArgs &a) {
    constexpr int E = 16 / sizeof(IN);
    const uint64_t lanes = (uint64_t)a.rows * (a.heads + 2 * a.kv_heads) * (D / 2 / E);
    hipLaunchKernelGGL((head_kernel<IN, OUT, KV, D, E>), dim3((uint32_t)((lanes + 255) / 256)), dim3(256), 0, ctx->stream, a);
}

template <typename IN, typename OUT, typename KV>
void launch_types(janus_ctx *ctx, const HeadArgs &a) {
    // the vector kernel reads and writes 16 bytes (8 of a binary16 output of binary32 rows) at a time
    const uintptr_t ptrs = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.kc |
                           (uintptr_t)a.vc | (uintptr_t)a.table | (uintptr_t)a.q_gamma | (uintptr_t)a.k_gamma;
    const bool aligned = (ptrs & 15u) == 0 && ((a.q_stride | a.k_stride | a.v_stride) * sizeof(IN) & 15u) == 0;
    if (aligned && a.hd == 64) launch_dim<IN, OUT, KV, 64>(ctx, a);
    else if (aligned && a.hd == 128) launch_dim<IN, OUT, KV, 128>(ctx, a);
    else if (aligned && a.hd == 256) launch_dim<IN, OUT, KV, 256>(ctx, a);
    else {
        const uint64_t heads = (uint64_t)a.rows * (a.heads + 2 * a.kv_heads);
        hipLaunchKernelGGL((head_any_kernel<IN, OUT, KV>), dim3((uint32_t)((heads + 3) / 4)), dim3(256), 0, ctx->stream, a);
    }
}

template <typename IN, typename OUT>
void launch_kv(janus_ctx *ctx, const HeadArgs &a, int kv_dt) {
    if (kv_dt == JANUS_DT_F16) launch_types<IN, OUT, _Float16>(ctx, a);
    else launch_types<IN, OUT, float>(ctx, a);
}

}  // namespace

int qk_norm_rope_launch(janus_ctx *ctx, const void *q, const void *k, const void *v, int in_dt, uint32_t q_stride,
                        uint32_t k_stride, uint32_t v_stride, const float *q_gamma, const float *k_gamma, float eps,
                        const float *table, void *q_out, int out_dt, void *kc, void *vc, int kv_dt, uint32_t rows,
                        uint32_t heads, uint32_t kv_heads, uint32_t hd, uint32_t position, uint32_t max_seq,
                        const int32_t *row_base, const int32_t *positions) {
    const HeadArgs a{q, k, v, q_stride, k_stride, v_stride, q_gamma, k_gamma, table, q_out, kc, vc,
                     row_base, positions, rows, heads, kv_heads, hd, position, max_seq, eps};
    if (in_dt == JANUS_DT_F16) {
        if (out_dt == JANUS_DT_F16) launch_kv<_Float16, _Float16>(ctx, a, kv_dt);
        else launch_kv<_Float16, float>(ctx, a, kv_dt);
    } else {
        if (out_dt == JANUS_DT_F16) launch_kv<float, _Float16>(ctx, a, kv_dt);
        else launch_kv<float, float>(ctx, a, kv_dt);
    }
    JANUS_LAUNCH_CHECK(ctx);
    return JANUS_OK;
}

}  // namespace janus
