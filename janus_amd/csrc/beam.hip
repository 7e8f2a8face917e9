// beam.hip -- beam search: the best continuations of each request's beams, and the
// caches that follow them.
//
// Selection. Token t of beam b has the value v = score_b + (x_t - L_b), L_b = log sum
// exp x; the n best of a request's beams x vocabulary are wanted, ties to the lowest
// index. Within a beam v goes by the logit, so one pass over the logits suffices:
//   select_part_kernel: a workgroup takes a part of a row (1024 logits a wavefront, in
//     registers), and keeps its maximum, its sum of exponentials and its n best logits.
//   select_join_kernel: a workgroup per request sums the parts to L_b and takes the n
//     best of all parts by v in binary64.
// The n best: the lanes' best values give a lower bound, found bit by bit with ballots;
// what is not below it, n values and a few more, is ranked by counting.
// Bound by the read of the logits: 16 requests of 8 beams, 128256 logits each, take 28 us (20
// for the first kernel, 3.2 TB/s, 8 for the second), one of 4 beams 14, the two launches.
// L_b is off by some 3e-8 (9e-8 at most over normal logits of sigma 0.5 to 6): the exponentials and sums of 16 of them are
// binary32, the sums of those binary64. Beams are compared by more than the last bits of their binary32 values.
//
// Reordering. Position by position the slots of a request's beams are permuted: a lane
// reads its bytes of every slot that is gone on from and then writes them to the
// slots that go on from it. Nothing else writes those bytes, so it works in place,
// without a copy of the cache and without a wait between workgroups. Bound by the read and write
// of what moves: four beams of 32 layers 91 us (4.6 TB/s), 64 beams 492 (4.95), where a
// large copy reaches 4.6.
#include <algorithm>
#include <cmath>

#include "internal.h"

namespace janus {
namespace {

constexpr uint32_t kPartWaves = 8;      // wavefronts of a part
constexpr uint32_t kLaneLogits = 16;    // logits of a lane, in groups of 4: all wavefronts of a CU fit (64 registers)
constexpr uint32_t kPart = kPartWaves * 64u * kLaneLogits;
constexpr uint32_t kJoinWaves = 8;
constexpr uint32_t kList = 1024;        // candidates that are ranked by counting
constexpr uint32_t kFew = 96;           // so many, and 8 n, are ranked without a look for a better bound
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

// A lower bound of the n-th largest of a wavefront's 64 keys (0 where fewer than n are not
// 0): the key bit by bit, until exactly n are left above.
__device__ __forceinline__ uint32_t nth_key(uint32_t key, uint32_t n) {
    uint32_t t = 0;
    for (int b = 31; b >= 0; --b) {
        const uint32_t at = t | 1u << b;
        const uint32_t have = (uint32_t)__popcll(__ballot(key >= at));
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

// e^t for t <= 0: log2 e in two parts, whose error would be common to all terms of a sum;
// the rounding of the product is not.
__device__ __forceinline__ float exp_neg(float t) {
    constexpr float kL = 1.44269502162933349609375f, kL2 = 1.92596299112661746887e-8f;   // log2 e = kL + kL2
    return __builtin_amdgcn_exp2f(fmaf(t, kL2, t * kL));
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
    __shared__ uint32_t share[kPartWaves];
    __shared__ float maxes[kPartWaves];
    __shared__ double sums[kPartWaves];
    __shared__ uint32_t found;
    __shared__ uint64_t best[2];
    const uint32_t row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
    if (a.scores && a.scores[row] == -INFINITY) return;   // an ended beam
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const float *x = a.logits + (size_t)row * a.vocab;
    // 1 KB for each wavefront in turn, so that all have their share of a short part too
    const uint32_t t0 = part * kPart + threadIdx.x * 4u;
    auto token = [&](uint32_t i) { return t0 + (i >> 2) * (kPartWaves * 256u) + (i & 3u); };
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
    float m = v[0];
#pragma unroll
    for (uint32_t i = 1; i < kLaneLogits; ++i) m = fmaxf(m, v[i]);
    // Each wavefront's n / 8-th best lane: the part has n values that are not below the least of the eight.
    const uint32_t key = t0 < a.vocab ? order32(m) : 0u;
    const uint32_t ks = nth_key(key, (a.n + kPartWaves - 1) / kPartWaves);
    if (lane == 0) share[wave] = ks;
    m = wave_max(m);
    // a NaN makes the sum a NaN, and so does +infinity by its difference to itself
    float s = 0.0f;
    if (m != -INFINITY) {
#pragma unroll
        for (uint32_t i = 0; i < kLaneLogits; ++i) s += exp_neg(v[i] - m);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kLaneLogits; ++i) s += v[i] != v[i] ? v[i] : 0.0f;
    }
    const double sum = wave_dsum((double)s);
    if (lane == 0) {
        maxes[wave] = m;
        sums[wave] = sum;
    }
    __syncthreads();
    uint32_t least = share[0];
#pragma unroll
    for (uint32_t w = 1; w < kPartWaves; ++w) least = min(least, share[w]);
    auto collect = [&]() {
        if (key && key >= least)
#pragma unroll
            for (uint32_t i = 0; i < kLaneLogits; ++i) {
                const uint32_t o = order32(v[i]);
                if (o >= least && token(i) < a.vocab) {
                    const uint32_t to = atomicAdd(&found, 1u);
                    if (to < kList) list[to] = (uint64_t)o << 32 | (uint32_t)~token(i);
                }
            }
        __syncthreads();
    };
    collect();
    if (found > max(kFew, 8u * a.n)) {
        // a wavefront without large values has kept the bound down, as in rows that leave some without any (3 beams of
        // 580 logits: 34 us where up to kList were ranked, 13 now): that of the n-th best lane of the best one
        __syncthreads();
        const uint32_t kn = nth_key(key, a.n);
        if (lane == 0) share[wave] = kn;
        if (threadIdx.x == 0) found = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < kPartWaves; ++w) least = max(least, share[w]);
        collect();
    }
    const size_t at = (size_t)row * a.parts + part;
    uint64_t *keys = a.keys + at * a.n;
    const uint32_t have = found;
    if (have <= kList) {
        for (uint32_t i = threadIdx.x; i < have; i += kPartWaves * 64u) {
            const uint64_t k = list[i];
            uint32_t rank = 0;
#pragma unroll 8
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
#pragma unroll
        for (uint32_t w = 1; w < kPartWaves; ++w) top = fmaxf(top, maxes[w]);
        double total = 0.0;
#pragma unroll
        for (uint32_t w = 0; w < kPartWaves; ++w)
            total += maxes[w] == -INFINITY ? sums[w] : sums[w] * (maxes[w] == top ? 1.0 : exp((double)maxes[w] - (double)top));
        a.part_max[at] = total != total ? __uint_as_float(0x7fc00000u) : top;
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
    __shared__ uint32_t share[kJoinWaves];
    __shared__ double lse[kMostBeams], score[kMostBeams];
    __shared__ int state[kMostBeams];
    __shared__ uint32_t found, deep;
    __shared__ Cand best[kJoinWaves];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row0 = blockIdx.x * a.beams;
    const uint32_t per_beam = a.parts * a.n, total = a.beams * per_beam;
    // the lane's first candidates are on their way while the sums are made (those of ended beams are whatever lies there)
    constexpr uint32_t kHeld = 8, kStep = kJoinWaves * 64u;
    // Where there are more than the lanes hold, the parts' best ones come first, then the second ones and so on: what is
    // not held is looked at only if a part's last held one is not below the bound. (8 requests of 16 beams, n 32: 26 us
    // for this kernel when all were, 17 now; 4 of 16, n 64: 96 and 20.)
    const uint32_t lists = a.beams * a.parts;
    const bool many = total > kHeld * kStep;
    auto place = [&](uint32_t c) { return many ? c % lists * a.n + c / lists : c; };
    uint64_t held[kHeld];
#pragma unroll
    for (uint32_t i = 0; i < kHeld; ++i) held[i] = threadIdx.x + i * kStep < total ? a.keys[(size_t)row0 * per_beam + place(threadIdx.x + i * kStep)] : 0ull;
    if (threadIdx.x == 0) found = deep = 0;
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
    auto value_of = [&](uint32_t c, uint64_t key) {
        const uint32_t b = c / per_beam, k = c - b * per_beam;
        if (state[b] != BEAM_FINE)   // all its tokens are alike: the first n stand for them
            return k < min(a.n, a.vocab) ? Cand{state[b] == BEAM_NAN ? ~0ull : order64(-INFINITY), b * a.vocab + k} : Cand{0, 0};
        if (!key) return Cand{0, 0};
        return Cand{order64(score[b] + ((double)value32((uint32_t)(key >> 32)) - lse[b])), b * a.vocab + (uint32_t)~key};
    };
    auto far = [&](uint32_t c) {   // beyond the held ones
        const uint32_t at = place(c);
        return value_of(at, a.keys[(size_t)row0 * per_beam + at]);
    };
    auto comes_before = [](const Cand &p, const Cand &q) { return p.hi > q.hi || (p.hi == q.hi && p.idx < q.idx); };
    Cand mine[kHeld];
    uint32_t top = 0;   // upper half of the lane's best
#pragma unroll
    for (uint32_t i = 0; i < kHeld; ++i) {
        mine[i] = threadIdx.x + i * kStep < total ? value_of(place(threadIdx.x + i * kStep), held[i]) : Cand{0, 0};
        top = max(top, (uint32_t)(mine[i].hi >> 32));
    }
    // as in the parts: the least of the wavefronts' shares, or else the best wavefront's n-th
    const uint32_t ks = nth_key(top, (a.n + kJoinWaves - 1) / kJoinWaves);
    if (lane == 0) share[wave] = ks;
    __syncthreads();
    uint32_t least = share[0];
#pragma unroll
    for (uint32_t w = 1; w < kJoinWaves; ++w) least = min(least, share[w]);
    auto collect = [&]() {
        auto take = [&](const Cand &k) {
            if (k.hi && (uint32_t)(k.hi >> 32) >= least) {
                const uint32_t to = atomicAdd(&found, 1u);
                if (to < kList) list[to] = k;
            }
        };
        if (top >= least) {
#pragma unroll
            for (uint32_t i = 0; i < kHeld; ++i) take(mine[i]);
        }
        if (many) {
            const uint32_t whole = kHeld * kStep / lists;   // held of every part
#pragma unroll
            for (uint32_t i = 0; i < kHeld; ++i)
                if ((uint32_t)(mine[i].hi >> 32) >= least && threadIdx.x + (i * kStep + lists) >= whole * lists) deep = 1;
            __syncthreads();
            if (deep)
                for (uint32_t c = threadIdx.x + kHeld * kStep; c < total; c += kStep) take(far(c));
        }
        __syncthreads();
    };
    collect();
    if (found > max(kFew, 8u * a.n)) {
        __syncthreads();
        const uint32_t kn = nth_key(top, a.n);
        if (lane == 0) share[wave] = kn;
        if (threadIdx.x == 0) found = deep = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < kJoinWaves; ++w) least = max(least, share[w]);
        collect();
    }
    const size_t at = (size_t)blockIdx.x * a.n;
    auto write = [&](uint32_t rank, const Cand &k) {
        const uint32_t b = k.idx / a.vocab;
        a.out[at + rank] = (float)value64(k.hi);
        a.parents[at + rank] = (int32_t)b;
        a.tokens[at + rank] = (int32_t)(k.idx - b * a.vocab);
    };
    const uint32_t have = found;
    if (have <= kList) {
        for (uint32_t i = threadIdx.x; i < have; i += kStep) {
            const Cand k = list[i];
            uint32_t rank = 0;
#pragma unroll 8
            for (uint32_t j = 0; j < have; ++j) rank += comes_before(list[j], k) ? 1u : 0u;
            if (rank < a.n) write(rank, k);
        }
    } else {
        Cand last{0, 0};
        for (uint32_t r = 0; r < a.n; ++r) {
            Cand next{0, 0xffffffffu};
            auto look = [&](const Cand &k) {
                if (k.hi && (r == 0 || comes_before(last, k)) && comes_before(k, next)) next = k;
            };
#pragma unroll
            for (uint32_t i = 0; i < kHeld; ++i) look(mine[i]);
            for (uint32_t c = threadIdx.x + kHeld * kStep; c < total; c += kStep) look(far(c));
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                const Cand k{(uint64_t)__shfl_xor((unsigned long long)next.hi, o, 64), (uint32_t)__shfl_xor((int)next.idx, o, 64)};
                if (comes_before(k, next)) next = k;
            }
            if (lane == 0) best[wave] = next;
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

// What a beam takes: `rows` rows from one slot to another. A beam that stays has 0, and
// the source of one that moves: its loads are made all the same (of lines that are there),
// so that no load waits behind a branch.
struct Move {
    uint32_t from, to, rows, rows_from;   // rows_from: rows that may be read at `from`
};

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// Vectors of a lane and beam at a time: 256 lanes move 16 KB of a slot in one go, or 8 where
// there are many beams. (64 beams of 32 layers, 2.4 GB: 492 us, 598 with one vector each.)
template <int B> constexpr uint32_t vectors_of() { return B <= 4 ? 4 : B <= 8 ? 2 : 1; }

template <typename V, int B> __device__ __forceinline__ void permute(char *base, uint64_t row, const Move *moves, uint32_t chunk, uint32_t chunks,
                                                                     uint32_t longest) {
    constexpr int U = vectors_of<B>();
    constexpr uint32_t kSpan = 256 * U * sizeof(V);
    for (uint64_t off = (uint64_t)chunk * kSpan; off < row * longest; off += (uint64_t)chunks * kSpan) {
        V v[B][U];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const uint64_t end = row * uniform(moves[i].rows_from) - sizeof(V);
#pragma unroll
            for (int u = 0; u < U; ++u)
                v[i][u] = *(const V *)(base + row * uniform(moves[i].from) + min(off + (threadIdx.x + 256 * u) * sizeof(V), end));
        }
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint64_t e = off + (threadIdx.x + 256 * u) * sizeof(V);
                if (e < row * uniform(moves[i].rows)) __builtin_nontemporal_store(v[i][u], (V *)(base + row * uniform(moves[i].to) + e));
            }
    }
}

template <int B> __global__ __launch_bounds__(256) void kv_reorder_kernel(ReorderArgs a) {
    __shared__ Move moves[B];
    const uint32_t chunk = blockIdx.x % a.chunks, unit = blockIdx.x / a.chunks;
    const uint32_t group = unit % a.groups, buf = unit / a.groups % a.bufs, layer = unit / a.groups / a.bufs;
    const uint32_t i = threadIdx.x & 63u;   // every wavefront finds the moves, the first one keeps them
    Move m{0, 0, 0, 0};
    if (i < B && i < a.beams) {
        const size_t g0 = (size_t)group * a.beams;
        const int32_t p = a.parents[g0 + i];
        if (p >= 0 && (uint32_t)p < a.beams && (uint32_t)p != i) {
            const int32_t from = a.row_base[g0 + p], to = a.row_base[g0 + i];
            int64_t n = a.seq_lens ? (int64_t)a.seq_lens[g0 + i] : (int64_t)a.max_seq;
            n = min(n, (int64_t)a.max_seq);
            n = min(n, (int64_t)a.cache_rows - max(from, to));
            if (from >= 0 && to >= 0 && from != to && n > 0) m = Move{(uint32_t)from, (uint32_t)to, (uint32_t)n, (uint32_t)n};
        }
    }
    const uint64_t some = __ballot(m.rows != 0);
    if (!some) return;
    const uint32_t one = (uint32_t)__builtin_ctzll(some);
    const uint32_t from = __shfl((int)m.from, one, 64), rows_from = __shfl((int)m.rows, one, 64);
    uint32_t longest = m.rows;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) longest = max(longest, (uint32_t)__shfl_xor((int)longest, o, 64));
    if (!m.rows) {
        m.from = from;
        m.rows_from = rows_from;
    }
    if (threadIdx.x < B) moves[threadIdx.x] = m;
    __syncthreads();
    char *base = a.buf[buf] + layer * a.layer_bytes[buf];
    longest = uniform(longest);
    if (a.vec[buf] == 16) permute<ju4, B>(base, a.row_bytes[buf], moves, chunk, a.chunks, longest);
    else if (a.vec[buf] == 4) permute<uint32_t, B>(base, a.row_bytes[buf], moves, chunk, a.chunks, longest);
    else permute<uint8_t, B>(base, a.row_bytes[buf], moves, chunk, a.chunks, longest);
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
    // enough workgroups for 64 on every CU, none without work where slots are full
    const uint64_t units = (uint64_t)layers * bufs * groups;
    const uint64_t want = std::max<uint64_t>(1, (uint64_t)ctx->num_cus * 64 / units);
    const uint64_t span = 256 * (beams <= 4 ? vectors_of<4>() : beams <= 8 ? vectors_of<8>() : vectors_of<16>());
    a.chunks = (uint32_t)std::min<uint64_t>(want, (most * max_seq + span - 1) / span);
    const dim3 grid((uint32_t)(units * a.chunks)), block(256);
    if (beams <= 4) hipLaunchKernelGGL((kv_reorder_kernel<4>), grid, block, 0, ctx->stream, a);
    else if (beams <= 8) hipLaunchKernelGGL((kv_reorder_kernel<8>), grid, block, 0, ctx->stream, a);
    else if (beams <= 16) hipLaunchKernelGGL((kv_reorder_kernel<16>), grid, block, 0, ctx->stream, a);
    else hipLaunchKernelGGL((kv_reorder_kernel<32>), grid, block, 0, ctx->stream, a);
    JANUS_LAUNCH_CHECK(ctx);
    return JANUS_OK;
}

}  // namespace janus
