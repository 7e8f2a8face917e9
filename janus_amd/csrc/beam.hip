// beam.hip -- beam search: the best continuations of each request's beams, and the
// caches that follow them.
//
// Selection. Token t of beam b has the value v = score_b + (x_t - L_b), L_b = log sum
// exp x; the n best of a request's beams x vocabulary are wanted, ties to the lowest
// index. Within a beam v goes by the logit, so one pass over the logits suffices:
//   select_part_kernel: a workgroup takes a part of a row (2048 logits a wavefront, in
//     registers), and keeps its maximum, its sum of exponentials and its n best logits.
//   select_join_kernel: a workgroup per request sums the parts to L_b and takes the n
//     best of all parts by v in binary64.
// The n best: the best of every 8 logits gives a lower bound (its n-th value, found bit
// by bit with ballots); what is not below it, n values and a few more, is ranked by
// counting.
// Bound by the read of the logits. L_b is kept to about 1e-8 (exponents in two parts,
// sums of many terms in binary64), so that beams are compared by more than the last
// bits of binary32.
//
// Reordering. Position by position the slots of a request's beams are permuted: a lane
// reads its 16 bytes of every slot that is gone on from and then writes them to the
// slots that go on from it. Nothing else touches those bytes, so it works in place,
// without a copy of the cache and without a wait.
#include <algorithm>
#include <cmath>

#include "internal.h"

namespace janus {
namespace {

constexpr uint32_t kPartWaves = 4;      // wavefronts of a part
constexpr uint32_t kLaneLogits = 32;    // logits of a lane, in groups of 8
constexpr uint32_t kPart = kPartWaves * 64u * kLaneLogits;
constexpr uint32_t kJoinWaves = 8;
constexpr uint32_t kList = 1024;        // candidates that are ranked by counting
constexpr uint32_t kMostBeams = 64;

// Order-preserving bits, never 0; zeros alike, NaN above all.
__device__ __forceinline__ uint32_t order32(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return v != v ? 0xffffffffu : (u >> 31 ? ~u : u | 0x80000000u);
}
__device__ __forceinline__ uint64_t order64(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
    return v != v ? ~0ull : (u >> 63 ? ~u : u | 0x8000000000000000ull);
}
__device__ __forceinline__ float value32(uint32_t k) { return __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ double value64(uint64_t k) {
    return k == ~0ull ? __longlong_as_double(0x7ff8000000000000ll) : __longlong_as_double((long long)(k >> 63 ? k ^ 0x8000000000000000ull : ~k));
}

// The n-th largest of a wavefront's 64 G keys, bit by bit; 0 where fewer than n are not 0.
// (Or a value below it with nothing in between: it stops where exactly n are left.)
template <int G> __device__ __forceinline__ uint32_t nth_key(const uint32_t (&key)[G], uint32_t n) {
    uint32_t t = 0;
    for (int b = 31; b >= 0; --b) {
        const uint32_t at = t | 1u << b;
        uint32_t have = 0;
#pragma unroll
        for (int i = 0; i < G; ++i) have += (uint32_t)__popcll(__ballot(key[i] >= at));
        if (have >= n) t = at;
        if (have == n) break;
    }
    return t;
}

__device__ __forceinline__ double wave_dsum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ uint64_t wave_umax(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint64_t)__shfl_xor((unsigned long long)v, o, 64));
    return v;
}

// e^t for t <= 0, off by about a step of binary32 (the product with log2 e in two parts).
__device__ __forceinline__ float exp_neg(float t) {
    constexpr float kL = 1.44269502162933349609375f, kL2 = 1.92596299112661746887e-8f;   // log2 e = kL + kL2
    const float hi = t * kL, lo = fmaf(t, kL, -hi) + t * kL2;
    const float e = __builtin_amdgcn_exp2f(hi);
    return t > -126.0f ? fmaf(e * 0.693147182f, lo, e) : e;   // t = -infinity has no second part
}

struct SelectArgs {
    const float *logits, *scores;
    float *out;
    int32_t *parents, *tokens;
    uint64_t *keys;            // [rows][parts][n] order32 << 32 | ~token, best first, 0: none
    float *part_max;           // [rows][parts]; NaN where a logit is NaN or +infinity
    double *part_sum;          // [rows][parts] of e^(x - maximum)
    uint32_t beams, vocab, n, parts;
};

template <bool VEC> __global__ __launch_bounds__(kPartWaves * 64) void select_part_kernel(SelectArgs a) {
    __shared__ uint64_t list[kList];
    __shared__ uint32_t nth[kPartWaves], share[kPartWaves];
    __shared__ float maxes[kPartWaves];
    __shared__ double sums[kPartWaves];
    __shared__ uint32_t found;
    __shared__ uint64_t best[2];
    const uint32_t row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    if (a.scores && a.scores[row] == -INFINITY) return;   // an ended beam
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const float *x = a.logits + (size_t)row * a.vocab;
    const uint32_t t0 = part * kPart + wave * (64u * kLaneLogits) + lane * 4u;
    auto token = [&](uint32_t i) { return t0 + (i >> 2) * 256u + (i & 3u); };
    if (threadIdx.x == 0) found = 0;
    float v[kLaneLogits];
#pragma unroll
    for (uint32_t i = 0; i < kLaneLogits; i += 4) {
        const uint32_t t = token(i);
        if (VEC) {
            const jf4 w = t < a.vocab ? __builtin_nontemporal_load((const jf4 *)(x + t)) : jf4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i + j] = w[j];
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) v[i + j] = t + j < a.vocab ? x[t + j] : -INFINITY;
        }
    }
    constexpr int G = kLaneLogits / 8;
    uint32_t key[G];   // the best of each group of 8
    float m = -INFINITY;
    bool odd = false;
#pragma unroll
    for (int k = 0; k < G; ++k) {
        float top = v[8 * k];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            top = fmaxf(top, v[8 * k + i]);
            odd |= !(v[8 * k + i] < INFINITY);
        }
        key[k] = token(8u * k) < a.vocab ? order32(top) : 0u;
        m = fmaxf(m, top);
    }
    m = wave_max(m);
    odd = __any(odd);
    float s = 0.0f;
    if (m != -INFINITY)
#pragma unroll
        for (uint32_t i = 0; i < kLaneLogits; ++i) s += exp_neg(v[i] - m);
    const double sum = wave_dsum((double)s);
    // n of the part's values are at least the n-th best group of any wavefront, and at least the n / kPartWaves-th of all
    const uint32_t kn = nth_key<G>(key, a.n), ks = nth_key<G>(key, (a.n + kPartWaves - 1) / kPartWaves);
    if (lane == 0) {
        nth[wave] = kn;
        share[wave] = ks;
        maxes[wave] = odd ? __uint_as_float(0x7fc00000u) : m;
        sums[wave] = sum;
    }
    __syncthreads();
    uint32_t least = share[0], some = nth[0];
#pragma unroll
    for (uint32_t w = 1; w < kPartWaves; ++w) {
        least = min(least, share[w]);
        some = max(some, nth[w]);
    }
    least = max(least, some);
#pragma unroll
    for (int k = 0; k < G; ++k)
        if (key[k] && key[k] >= least)
#pragma unroll
            for (uint32_t i = 8 * k; i < 8u * (k + 1); ++i) {
                const uint32_t o = order32(v[i]);
                if (o >= least && token(i) < a.vocab) {
                    const uint32_t to = atomicAdd(&found, 1u);
                    if (to < kList) list[to] = (uint64_t)o << 32 | (uint32_t)~token(i);
                }
            }
    __syncthreads();
    const size_t at = (size_t)row * a.parts + part;
    uint64_t *keys = a.keys + at * a.n;
    const uint32_t have = found;
    if (have <= kList) {
        for (uint32_t i = threadIdx.x; i < have; i += kPartWaves * 64u) {
            const uint64_t k = list[i];
            uint32_t rank = 0;
            for (uint32_t j = 0; j < have; ++j) rank += list[j] > k ? 1u : 0u;
            if (rank < a.n) keys[rank] = k;
        }
        for (uint32_t i = have + threadIdx.x; i < a.n; i += kPartWaves * 64u) keys[i] = 0;
    } else {
        // masses of equal logits: the next best one n times
        uint64_t last = ~0ull;
        for (uint32_t r = 0; r < a.n; ++r) {
            if (threadIdx.x == 0) best[r & 1u] = 0;
            __syncthreads();
            uint64_t mine = 0;
#pragma unroll
            for (uint32_t i = 0; i < kLaneLogits; ++i) {
                const uint64_t k = token(i) < a.vocab ? (uint64_t)order32(v[i]) << 32 | (uint32_t)~token(i) : 0ull;
                if (k < last) mine = max(mine, k);
            }
            mine = wave_umax(mine);
            if (lane == 0) atomicMax((unsigned long long *)&best[r & 1u], (unsigned long long)mine);
            __syncthreads();
            last = best[r & 1u];
            if (threadIdx.x == 0) keys[r] = last;
        }
    }
    if (threadIdx.x == 0) {
        float top = maxes[0];
        bool nan = top != top;
        for (uint32_t w = 1; w < kPartWaves; ++w) {
            nan |= maxes[w] != maxes[w];
            top = fmaxf(top, maxes[w]);
        }
        double total = 0.0;
        for (uint32_t w = 0; w < kPartWaves; ++w)
            if (maxes[w] > -INFINITY) total += sums[w] * exp((double)maxes[w] - (double)top);
        a.part_max[at] = nan ? __uint_as_float(0x7fc00000u) : top;
        a.part_sum[at] = total;
    }
}

enum { BEAM_FINE = 0, BEAM_NAN = 1, BEAM_ENDED = 2 };

struct Cand {
    uint64_t hi;    // order64 of the value; 0: none
    uint32_t idx;   // beam * vocab + token
};

__global__ __launch_bounds__(kJoinWaves * 64) void select_join_kernel(SelectArgs a) {
    __shared__ Cand list[kList];
    __shared__ uint32_t nth[kJoinWaves], share[kJoinWaves];
    __shared__ double lse[kMostBeams], score[kMostBeams];
    __shared__ int state[kMostBeams];
    __shared__ uint32_t found;
    __shared__ Cand best[kJoinWaves];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row0 = blockIdx.x * a.beams;
    if (threadIdx.x == 0) found = 0;
    for (uint32_t b = wave; b < a.beams; b += kJoinWaves) {
        const float sc = a.scores ? a.scores[row0 + b] : 0.0f;
        int st = sc == -INFINITY ? BEAM_ENDED : (sc < INFINITY ? BEAM_FINE : BEAM_NAN);
        double l = 0.0;
        if (st == BEAM_FINE) {
            const size_t at = (size_t)(row0 + b) * a.parts;
            float top = -INFINITY;
            bool nan = false;
            for (uint32_t i = lane; i < a.parts; i += 64) {
                const float m = a.part_max[at + i];
                nan |= m != m;
                top = fmaxf(top, m);
            }
            top = wave_max(top);
            if (__any(nan)) st = BEAM_NAN;
            else if (top == -INFINITY) st = BEAM_ENDED;
            else {
                double s = 0.0;
                for (uint32_t i = lane; i < a.parts; i += 64) {
                    const float m = a.part_max[at + i];
                    if (m != -INFINITY) s += a.part_sum[at + i] * exp((double)m - (double)top);
                }
                l = (double)top + log(wave_dsum(s));
            }
        }
        if (lane == 0) {
            lse[b] = l;
            score[b] = (double)sc;
            state[b] = st;
        }
    }
    __syncthreads();
    const uint32_t per_beam = a.parts * a.n, total = a.beams * per_beam;
    auto get = [&](uint32_t c) {
        const uint32_t b = c / per_beam, k = c % per_beam;
        if (state[b] != BEAM_FINE)   // all its tokens are alike: the first n stand for them
            return k < min(a.n, a.vocab) ? Cand{state[b] == BEAM_NAN ? ~0ull : order64(-INFINITY), b * a.vocab + k} : Cand{0, 0};
        const uint64_t key = a.keys[(size_t)(row0 + b) * per_beam + k];
        if (!key) return Cand{0, 0};
        return Cand{order64(score[b] + ((double)value32((uint32_t)(key >> 32)) - lse[b])), b * a.vocab + (uint32_t)~key};
    };
    auto comes_before = [](const Cand &p, const Cand &q) { return p.hi > q.hi || (p.hi == q.hi && p.idx < q.idx); };
    uint32_t top[1] = {0};   // upper half of the lane's best
    for (uint32_t c = threadIdx.x; c < total; c += kJoinWaves * 64u) top[0] = max(top[0], (uint32_t)(get(c).hi >> 32));
    const uint32_t kn = nth_key<1>(top, a.n), ks = nth_key<1>(top, (a.n + kJoinWaves - 1) / kJoinWaves);
    if (lane == 0) {
        nth[wave] = kn;
        share[wave] = ks;
    }
    __syncthreads();
    uint32_t least = share[0], some = nth[0];
#pragma unroll
    for (uint32_t w = 1; w < kJoinWaves; ++w) {
        least = min(least, share[w]);
        some = max(some, nth[w]);
    }
    least = max(least, some);
    for (uint32_t c = threadIdx.x; c < total; c += kJoinWaves * 64u) {
        const Cand k = get(c);
        if (k.hi && (uint32_t)(k.hi >> 32) >= least) {
            const uint32_t to = atomicAdd(&found, 1u);
            if (to < kList) list[to] = k;
        }
    }
    __syncthreads();
    const size_t at = (size_t)blockIdx.x * a.n;
    auto write = [&](uint32_t rank, const Cand &k) {
        a.out[at + rank] = (float)value64(k.hi);
        a.parents[at + rank] = (int32_t)(k.idx / a.vocab);
        a.tokens[at + rank] = (int32_t)(k.idx % a.vocab);
    };
    const uint32_t have = found;
    if (have <= kList) {
        for (uint32_t i = threadIdx.x; i < have; i += kJoinWaves * 64u) {
            const Cand k = list[i];
            uint32_t rank = 0;
            for (uint32_t j = 0; j < have; ++j) rank += comes_before(list[j], k) ? 1u : 0u;
            if (rank < a.n) write(rank, k);
        }
    } else {
        Cand last{0, 0};
        for (uint32_t r = 0; r < a.n; ++r) {
            Cand mine{0, 0xffffffffu};
            for (uint32_t c = threadIdx.x; c < total; c += kJoinWaves * 64u) {
                const Cand k = get(c);
                if (k.hi && (r == 0 || comes_before(last, k)) && comes_before(k, mine)) mine = k;
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                const Cand k{(uint64_t)__shfl_xor((unsigned long long)mine.hi, o, 64), (uint32_t)__shfl_xor((int)mine.idx, o, 64)};
                if (comes_before(k, mine)) mine = k;
            }
            if (lane == 0) best[wave] = mine;
            __syncthreads();
            last = best[0];
#pragma unroll
            for (uint32_t w = 1; w < kJoinWaves; ++w)
                if (comes_before(best[w], last)) last = best[w];
            if (threadIdx.x == 0) write(r, last);
            __syncthreads();
        }
    }
}

// ---- reordering ---------------------------------------------------------------

constexpr uint32_t kMostBufs = JANUS_REORDER_BUFFERS;

struct ReorderArgs {
    char *buf[kMostBufs];
    uint64_t row_bytes[kMostBufs], layer_bytes[kMostBufs];
    uint32_t vec[kMostBufs];           // bytes that a lane moves at a time: 16, 4 or 1
    const int32_t *row_base, *parents, *seq_lens;
    uint32_t bufs, groups, beams, cache_rows, max_seq, chunks;
};

struct Move {
    uint64_t from, to;   // rows
    uint32_t rows;
};

template <typename V, int B> __device__ __forceinline__ void permute(char *base, uint64_t row_bytes, const Move *moves, uint32_t chunk, uint32_t chunks,
                                                                     uint32_t longest) {
    V *const at = (V *)base;
    const uint64_t row = row_bytes / sizeof(V), end = row * longest;
    for (uint64_t e = (uint64_t)chunk * 256u + threadIdx.x; e < end; e += (uint64_t)chunks * 256u) {
        V v[B];
#pragma unroll
        for (int i = 0; i < B; ++i)
            if (e < moves[i].rows * row) v[i] = at[moves[i].from * row + e];
#pragma unroll
        for (int i = 0; i < B; ++i)
            if (e < moves[i].rows * row) at[moves[i].to * row + e] = v[i];
    }
}

template <int B> __global__ __launch_bounds__(256) void kv_reorder_kernel(ReorderArgs a) {
    __shared__ Move moves[B];
    __shared__ uint32_t longest;
    const uint32_t chunk = blockIdx.x % a.chunks, unit = blockIdx.x / a.chunks;
    const uint32_t group = unit % a.groups, buf = unit / a.groups % a.bufs, layer = unit / a.groups / a.bufs;
    if (threadIdx.x == 0) longest = 0;
    __syncthreads();
    if (threadIdx.x < B) {
        Move m{0, 0, 0};
        const uint32_t i = threadIdx.x;
        if (i < a.beams) {
            const size_t g0 = (size_t)group * a.beams;
            const int32_t p = a.parents[g0 + i];
            if (p >= 0 && (uint32_t)p < a.beams && (uint32_t)p != i) {
                const int64_t from = a.row_base[g0 + p], to = a.row_base[g0 + i];
                int64_t n = a.seq_lens ? (int64_t)a.seq_lens[g0 + i] : (int64_t)a.max_seq;
                n = min(n, (int64_t)a.max_seq);
                n = min(n, (int64_t)a.cache_rows - max(from, to));
                if (from >= 0 && to >= 0 && from != to && n > 0) m = Move{(uint64_t)from, (uint64_t)to, (uint32_t)n};
            }
        }
        moves[i] = m;
        if (m.rows) atomicMax(&longest, m.rows);
    }
    __syncthreads();
    const uint32_t n = longest;
    if (!n) return;
    char *base = a.buf[buf] + layer * a.layer_bytes[buf];
    if (a.vec[buf] == 16) permute<ju4, B>(base, a.row_bytes[buf], moves, chunk, a.chunks, n);
    else if (a.vec[buf] == 4) permute<uint32_t, B>(base, a.row_bytes[buf], moves, chunk, a.chunks, n);
    else permute<uint8_t, B>(base, a.row_bytes[buf], moves, chunk, a.chunks, n);
}

}  // namespace

int beam_select_launch(janus_ctx *ctx, const float *logits, const float *scores, float *out, int32_t *parents,
                       int32_t *tokens, uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t n) {
    SelectArgs a{};
    a.logits = logits;
    a.scores = scores;
    a.out = out;
    a.parents = parents;
    a.tokens = tokens;
    a.beams = beams;
    a.vocab = vocab;
    a.n = n;
    a.parts = (vocab + kPart - 1) / kPart;
    const size_t cells = (size_t)batch * beams * a.parts;
    if (int e = ensure_gemm_ws(ctx, cells * (n * 8 + 12))) return e;
    a.keys = (uint64_t *)ctx->gemm_ws;
    a.part_sum = (double *)(a.keys + cells * n);
    a.part_max = (float *)(a.part_sum + cells);
    const dim3 grid((uint32_t)cells), block(kPartWaves * 64);
    if (vocab % 4 == 0 && ((uintptr_t)logits & 15u) == 0) hipLaunchKernelGGL((select_part_kernel<true>), grid, block, 0, ctx->stream, a);
    else hipLaunchKernelGGL((select_part_kernel<false>), grid, block, 0, ctx->stream, a);
    JANUS_LAUNCH_CHECK(ctx);
    hipLaunchKernelGGL(select_join_kernel, dim3(batch), dim3(kJoinWaves * 64), 0, ctx->stream, a);
    JANUS_LAUNCH_CHECK(ctx);
    return JANUS_OK;
}

int kv_reorder_launch(janus_ctx *ctx, uint32_t bufs, void *const *buf, const uint64_t *row_bytes, uint32_t layers,
                      uint32_t groups, uint32_t beams, uint32_t cache_rows, uint32_t max_seq, const int32_t *row_base,
                      const int32_t *parents, const int32_t *seq_lens) {
    ReorderArgs a{};
    uint64_t most = 1;
    for (uint32_t i = 0; i < bufs; ++i) {
        a.buf[i] = (char *)buf[i];
        a.row_bytes[i] = row_bytes[i];
        a.layer_bytes[i] = row_bytes[i] * cache_rows;
        const uint64_t all = (uint64_t)(uintptr_t)buf[i] | row_bytes[i];   // layers are whole rows apart
        a.vec[i] = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
        most = std::max(most, row_bytes[i] / a.vec[i]);
    }
    a.row_base = row_base;
    a.parents = parents;
    a.seq_lens = seq_lens;
    a.bufs = bufs;
    a.groups = groups;
    a.beams = beams;
    a.cache_rows = cache_rows;
    a.max_seq = max_seq;
    const uint64_t units = (uint64_t)layers * bufs * groups;
    const uint64_t want = std::max<uint64_t>(1, (uint64_t)ctx->num_cus * 16 / units);
    a.chunks = (uint32_t)std::min<uint64_t>(want, (most * max_seq + 255) / 256);
    const dim3 grid((uint32_t)(units * a.chunks)), block(256);
    if (beams <= 4) hipLaunchKernelGGL((kv_reorder_kernel<4>), grid, block, 0, ctx->stream, a);
    else if (beams <= 8) hipLaunchKernelGGL((kv_reorder_kernel<8>), grid, block, 0, ctx->stream, a);
    else if (beams <= 16) hipLaunchKernelGGL((kv_reorder_kernel<16>), grid, block, 0, ctx->stream, a);
    else hipLaunchKernelGGL((kv_reorder_kernel<32>), grid, block, 0, ctx->stream, a);
    JANUS_LAUNCH_CHECK(ctx);
    return JANUS_OK;
}

}  // namespace janus
