// packed.hip -- attention of packed rows over the KV cache: causal attention of
// the prompts, chunks and drafted tokens of several requests in one launch, and
// decode attention of a batch behind a shared prefix.
//
// The queries of a KV head that read the same K and V are the columns of one
// matrix product: column c of a sequence of n rows is query head c % G of its
// row c / G (G heads per KV head), so few rows of many heads fill a tile as many
// rows of few heads do, and K and V are read once for all of them. A workgroup
// takes up to 128 columns, passes over the positions and keeps the running maximum
// m, the sum l and the output O^T in registers:
//   S^T = K Q^T (positions x columns), p = 2^(scale log2(e) (s - m)),
//   l <- l 2^(m_old - m) + sum p,  O^T <- O^T 2^(m_old - m) + V^T P^T.
// A lane's column is one query, so m, l and the rescale are per lane, and P is
// the second product's operand as it lies; V's operand in binary16 is read from LDS
// with the transposing load in the position order that matches.
//   binary16 rows and cache: f16 MFMAs, P rounded to binary16 (its errors average
//     out over the positions and stay below the output's own rounding);
//   binary32 rows, binary16 cache: q and P in two binary16 parts each (22 bits);
//   binary32 rows and cache: f32 MFMAs, nothing rounded.
// m follows the maximum only when that would grow by more than a few powers of
// two (an exponent bias leaves P room), so most tiles rescale nothing.
//
// wide_tile (on a binary16 cache 33 columns and more, in two parts 17, and fewer on
// split contexts) shares K and V through LDS; few_columns (the others) gives every
// wavefront positions of its own.
//
// Few columns on a long context: the positions are split over workgroups, each
// of which writes (m, l) and its output, and a second launch joins them. A
// shared prefix is a sequence of its own with one row per request and no causal
// limit; its parts and those of the requests' own positions are joined alike.
//
// Measured (32/8/128 heads, binary16 unless named, the launches of a call back to
// back, here and below): a prompt of 8192 rows 558 us, 985 TFLOP/s (a large matrix
// product reaches 1050); 24 prompts of 3 to 700 rows 72 us (174 MB, 34 GFLOP); the last
// 512 binary32 rows of 8192 on a binary16 cache 142 us (67 GFLOP twice, for the two
// parts); six prompts of 33 to 512 rows at 32/32/128 in binary32 67 us (4.5 GFLOP; 121
// TFLOP/s on long ones); five drafted tokens each of 16 requests 34 us (137 MB); 64
// binary32 rows behind 16384 positions 68 us (206 MB).
#include <algorithm>

#include "internal.h"

namespace janus {
namespace {

typedef _Float16 ph8 __attribute__((ext_vector_type(8)));
typedef short ps4 __attribute__((ext_vector_type(4)));
typedef float pf4 __attribute__((ext_vector_type(4)));
typedef float pf16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) ps4 *lds4;

struct PackedArgs {
    const void *q;            // [rows][heads][D]
    const void *kc, *vc;      // [cache rows][kv_heads][D]
    void *out;                // [rows][heads][D]
    float *part;              // split: [rows][heads][slots][D], then (m, l) [rows][heads][slots][2]
    float *part_ml;
    const int32_t *q_start;   // [nseq + 1], or null: rows / nseq rows each
    const int32_t *row_base;  // null: s * max_seq
    const int32_t *seq_lens;  // null: seq_len, or as many as the sequence has rows
    uint32_t rows, nseq, heads, kv_heads, G;
    uint32_t cols;            // columns per workgroup: 16 to 128, a power of two
    uint32_t max_seq;
    int64_t seq_len;          // < 0: the rows
    uint32_t splits;          // most parts of a tile's positions (1: never split)
    uint32_t target;          // parts per KV head to aim at
    uint32_t slots;           // partials per row and head (0: results are written)
    uint32_t prefix_row, prefix_len, prefix_tiles, prefix_splits;
    uint32_t prefix_blocks;   // workgroups of the prefix, before the others
    uint32_t longest;         // 1: tiles by the position that they reach
    uint32_t light;           // 1: the Light kernel
    float scale2;             // scale * log2(e)
};

// What a workgroup works on.
struct Work {
    uint32_t row0, n;         // rows of the sequence (of the batch, for a prefix)
    uint32_t c0;              // first column
    size_t kv_row;            // cache row of position 0
    uint32_t len;             // positions that there are
    int32_t first;            // of those, row 0 sees so many (below 1: none) and each row one more than the last
    bool causal;              // else every row sees all
    uint32_t part, parts, chunk, slot;   // positions [part chunk, + chunk); slot of the partials
};

// The maximum over all lanes, without LDS traffic.
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));   // row_ror:8, 4, 2, 1
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
    return max(max((uint32_t)__builtin_amdgcn_readlane(v, 0), (uint32_t)__builtin_amdgcn_readlane(v, 16)),
               max((uint32_t)__builtin_amdgcn_readlane(v, 32), (uint32_t)__builtin_amdgcn_readlane(v, 48)));
}

// Rows [first, first + n), first cache row and positions of sequence s. Whatever
// the tables hold, rows stay inside [0, rows) and positions within [0, max_seq].
__device__ __forceinline__ void sequence_of(const PackedArgs &a, uint32_t s, Work &w) {
    const int64_t base = a.row_base ? (int64_t)a.row_base[s] : (int64_t)s * a.max_seq;
    const int32_t given = a.seq_lens ? a.seq_lens[s] : 0;
    if (a.q_start) {
        const int32_t b = a.q_start[s], e = a.q_start[s + 1], lim = (int32_t)a.rows;
        const int32_t first = min(max(b, 0), lim);
        w.row0 = (uint32_t)first;
        w.n = (uint32_t)(min(max(e, first), lim) - first);
    } else {
        w.n = a.rows / a.nseq;
        w.row0 = s * w.n;
    }
    const uint32_t len = a.seq_lens ? (uint32_t)max(given, 0) : a.seq_len < 0 ? w.n : (uint32_t)a.seq_len;   // below 2^31
    w.len = base < 0 ? 0u : min(len, a.max_seq);
    w.first = (int32_t)(len + 1u - w.n);   // n > 0 wherever it is used
    w.kv_row = base < 0 ? 0 : (size_t)base;
}

// The sequence, tile and part of task t; false: there is none. A sequence's tiles
// go from its last to its first.
//
// Splitting (few tiles): the tables give the positions of all tiles, and every part
// gets as many, so that long and short contexts take equal workgroups. Every workgroup
// finds the same numbers.
//
// With `longest`, the tiles of all sequences go by the position that they reach, the
// farthest first, so that no long one is begun when the others are done; else the
// sequences follow each other, which keeps their K and V in L2. Binary32 caches take
// the former, where a position costs 16 times the matrix time (six prompts of 33 to 512
// rows at 32/32/128: 67 us against 86; 20 of 3 to 69 behind up to 85 positions: 37
// against 35); binary16 caches the latter (24 prompts of 3 to 700 rows at 32/8/128: 70
// us either way; binary32 rows on them: 117 either way, 20 of 3 to 69 rows at 32/32/128
// 18.6 against 19.9, six of 31 to 633 at 40/8/128 48 against 47).
__device__ __forceinline__ bool find_task(const PackedArgs &a, uint32_t t, Work &w) {
    const uint32_t lane = threadIdx.x & 63u, shift = 31u - __builtin_clz(a.cols);
    w.causal = true;
    w.part = 0;
    w.parts = 1;
    w.chunk = 0x80000000u;
    if (!a.q_start && a.splits == 1) {
        const uint32_t each = (a.rows / a.nseq * a.G + a.cols - 1) >> shift, s = t / each;
        if (s >= a.nseq) return false;
        sequence_of(a, s, w);
        w.c0 = (each - 1 - t % each) << shift;
        return true;
    }
    // a lane per sequence; tiles of it
    Work x;
    auto sequence = [&](uint32_t s0) -> uint32_t {
        sequence_of(a, min(s0 + lane, a.nseq - 1), x);
        return s0 + lane < a.nseq ? (x.n * a.G + a.cols - 1) >> shift : 0u;   // n G < 2^25
    };
    auto take = [&](int at, uint32_t tile) {
        auto pick = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane(v, at); };
        w.row0 = pick(x.row0);
        w.n = pick(x.n);
        w.len = pick(x.len);
        w.first = (int32_t)pick((uint32_t)x.first);
        w.kv_row = pick((uint32_t)x.kv_row);   // below 2^31
        w.c0 = tile << shift;
        return true;
    };
    uint32_t mine = sequence(0);
    if (a.longest) {   // at most 64 sequences, not split
        // levels: a tile's distance from position 0 in tiles; lane j counts those from lo + j step on
        const uint32_t before = x.len > x.n ? (uint32_t)min((uint64_t)(x.len - x.n) * a.G >> shift, (uint64_t)1 << 30) : 0u;
        const uint32_t top = before + mine;
        const uint32_t most = max_dpp(mine ? top : 0u);
        uint32_t lo = 0, above = 0;   // level of task t, tiles above it
        for (uint32_t step = 1u << max(0, 26 - (int)__builtin_clz(most | 1u));; step = step > 64 ? step >> 6 : 1) {
            const uint32_t level = lo + lane * step;
            uint32_t count = 0;
            for (uint32_t s = 0; s < a.nseq; ++s)
                count += (uint32_t)min(max((int32_t)(__builtin_amdgcn_readlane(top, s) - level), 0), (int32_t)__builtin_amdgcn_readlane(mine, s));
            const uint64_t hit = __ballot(count > t);   // the first lanes: count falls with the level
            if (!hit) return false;
            const int at = 63 - __builtin_clzll(hit);
            lo = __builtin_amdgcn_readlane(level, at);
            if (at < 63) above = __builtin_amdgcn_readlane(count, at + 1);   // else as found with the longer step
            if (step == 1) break;
        }
        uint64_t has = __ballot(mine && before <= lo && lo < top);
        for (uint32_t r = t - above; r; --r) has &= has - 1;
        const int at = __ffsll((unsigned long long)has) - 1;
        return take(at, lo - __builtin_amdgcn_readlane(before, at));
    }
    if (a.splits > 1) {
        float total = 0.0f;
        uint32_t longest = 0;
        for (uint32_t s0 = 0; s0 < a.nseq; s0 += 64) {
            const uint32_t tiles = s0 ? sequence(s0) : mine;
            total += (float)tiles * (float)x.len;
            longest = max(longest, tiles ? x.len : 0u);
        }
        total = wave_sum_dpp(total);
        longest = max_dpp(longest);
        const uint32_t even = (uint32_t)fminf(total / (float)a.target, 1e9f) + 1, least = (longest + a.splits - 1) / a.splits;
        w.chunk = __builtin_amdgcn_readfirstlane((max(max(even, least), 128u) + 63u) / 64u * 64u);
        if (a.nseq > 64) mine = sequence(0);
    }
    for (uint32_t s0 = 0;;) {
        const uint32_t parts = max((x.len + w.chunk - 1) / w.chunk, 1u), tasks = mine * parts;
        const uint32_t upto = scan_dpp(tasks);
        const uint64_t hit = __ballot(t < upto);
        if (hit) {
            const int at = __ffsll((unsigned long long)hit) - 1;
            const uint32_t r = t - __builtin_amdgcn_readlane(upto - tasks, at);
            w.parts = __builtin_amdgcn_readlane(parts, at);
            w.part = r % w.parts;
            return take(at, __builtin_amdgcn_readlane(mine, at) - 1 - r / w.parts);
        }
        t -= __builtin_amdgcn_readlane(upto, 63);
        if ((s0 += 64) >= a.nseq) return false;
        mine = sequence(s0);
    }
}

// Positions that row i of the work sees: all, or first + i of them, which is at most
// the sequence's own length and may be more than there are (max_seq_len is shorter).
__device__ __forceinline__ uint32_t seen_of(const Work &w, uint32_t i) {
    return w.causal ? min((uint32_t)max(w.first + (int32_t)i, 0), w.len) : w.len;
}

// LDS of a tile of TP positions: K rows, then V rows, 16-byte segments permuted
// within a row so that the reads below meet each bank as rarely as they can: 32
// lanes read a segment of 32 rows of K, 16 lanes 32 bytes of each of 4 rows of V
// (transposing read).
template <int D> struct Lay {
    static constexpr uint32_t RB = D * 2, SEGS = RB / 16;
    static __device__ __forceinline__ uint32_t k_swz(uint32_t row) {
        return SEGS >= 16 ? (row & 15u) : (((row >> 1) & 7u) ^ ((row & 1u) << 2));
    }
    static __device__ __forceinline__ uint32_t v_swz(uint32_t row) {
        return SEGS >= 16 ? (row & 3u) << 2 : ((row >> 1) & 1u) << 2;
    }
    // few columns: 64 lanes read 32 bytes of each of 16 rows of V
    static __device__ __forceinline__ uint32_t few_swz(uint32_t row) {
        return SEGS >= 16 ? (row & 7u) << 1 : ((row >> 1) & 3u) << 1;
    }
};

// p carries 2^BIAS; m may lag behind the maximum by 2^SLACK (p stays below 2^16
// where it becomes binary16)
template <typename Q, typename KV> struct Range {
    static constexpr bool H = sizeof(KV) == 2, TWO = H && sizeof(Q) == 4;   // TWO: q and P in two parts
    static constexpr float BIAS = !H ? 0.0f : TWO ? 13.0f : 6.0f, SLACK = TWO ? 2.0f : 8.0f;
};

// Sum that is NaN exactly if the 16 bytes hold an infinity or NaN.
template <typename KV> __device__ __forceinline__ float odd_sum(const ju4 &v, float s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(KV) == 2) s = __builtin_amdgcn_fdot2(__builtin_bit_cast(jh2, (uint32_t)v[i]), (jh2)(_Float16)0.0f, s, false);
        else s = fmaf(__uint_as_float(v[i]), 0.0f, s);
    }
    return s;
}

// The finite values of the 16 bytes, others as 0.
template <typename KV> __device__ __forceinline__ ju4 finite_part(ju4 v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(KV) == 2) {
            if ((v[i] & 0x7c00u) == 0x7c00u) v[i] &= 0xffff0000u;
            if ((v[i] & 0x7c000000u) == 0x7c000000u) v[i] &= 0xffffu;
        } else if ((v[i] & 0x7f800000u) == 0x7f800000u) {
            v[i] = 0u;
        }
    }
    return v;
}

// Most columns that few_columns takes on a binary16 cache (two column tiles of
// two-part q and P would not fit the registers).
template <typename Q, typename KV> constexpr uint32_t few_of() { return Range<Q, KV>::TWO ? 16u : 32u; }

// 2^sh that takes the largest of the elements to 2^14 .. 2^15 (below 2^-85 no
// score counts), so that two binary16 parts hold 22 bits of it, and of the others
// down to 2^-39 of it.
__device__ __forceinline__ float two_part_scale(float qmax) {
    int qe = 0;
    (void)frexpf(qmax, &qe);
    return ldexpf(1.0f, -max(qe - 15, -100));
}

// Results of up to 16 NT CW columns and the positions [p0, p1), no barrier on the
// way: the wavefronts are CW groups of columns (1 or 2) by 4 / CW of positions; those
// of a group take steps of positions in turn, each reading its own K and V, and are
// joined through LDS. A column is a lane of 16; NT column tiles share the operands.
//   S^T [16 positions x 16 columns]: lane 16 g + i holds positions 4 g + v of
//   column i. K comes from memory as the operand: position i, its dims by g.
//   binary16: steps of 32 positions (two S^T), v_mfma_f32_16x16x32_f16; V through
//     LDS and the transposing read, dims 16 d + 4 g + v of column i in o[d];
//   binary32: steps of 16, v_mfma_f32_16x16x4_f32 with k = g the position 4 g + v,
//     so V is the operand as loaded: dims 4 (i + 16 e) + c in tile 4 e + c, and
//     o[4 e + c] holds dims 4 (4 g + v + 16 e) + c.
template <typename Q, typename KV, int D, int NT>
__device__ __forceinline__ void few_columns(const PackedArgs &a, const Work &w, uint32_t kvh, uint32_t ncols,
                                            uint32_t p0, uint32_t p1, uint32_t cw, unsigned char *smem) {
    typedef Range<Q, KV> R;
    typedef Lay<D> Y;
    constexpr bool H = R::H, TWO = R::TWO;
    constexpr int STEP = H ? 32 : 16, NB = STEP / 16;
    constexpr int KS = H ? D / 32 : D / 16;          // 16-byte loads of K per position tile
    constexpr int VS = STEP * D * (int)sizeof(KV) / 1024;   // 16-byte loads of V per step
    constexpr int ND = D / 16;
    constexpr uint32_t RB = D * sizeof(KV);
    uint32_t tid = threadIdx.x;
    asm volatile("" : "+v"(tid));   // what follows from it stays out of the code before, which may need the registers
    const uint32_t lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t i = lane & 15u, g = lane >> 4;
    const uint32_t pw = 4u / cw, cg = wave & (cw - 1u), pg = wave / cw;   // this wavefront's columns and positions
    const uint32_t c0 = w.c0 + 16u * NT * cg;
    const uint32_t kvrow = a.kv_heads * RB;          // bytes from a position to the next
    const unsigned char *kc = (const unsigned char *)a.kc + (w.kv_row * a.kv_heads + kvh) * RB;
    const unsigned char *vc = (const unsigned char *)a.vc + (w.kv_row * a.kv_heads + kvh) * RB;

    // the positions that this wavefront's columns see at all
    const uint32_t e1 = c0 < ncols ? min(seen_of(w, min(c0 + 16u * NT - 1, ncols - 1) / a.G), p1) : 0u;
    ju4 kr[NB][KS], vr[VS];
    auto load_k = [&](uint32_t p) {
        const unsigned char *at = kc + (size_t)p * kvrow;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int t = 0; t < KS; ++t)
                kr[b][t] = *(const ju4 *)(at + (min(16u * b + i, e1 - 1 - p) * kvrow + (4u * t + g) * 16u));
    };
    auto load_v = [&](uint32_t p) {
        const unsigned char *at = vc + (size_t)p * kvrow;
#pragma unroll
        for (int j = 0; j < VS; ++j) {
            // binary16: in order; binary32: position 4 g + j / E, segment i + 16 (j % E)
            constexpr int E = D / 64;
            const uint32_t s = lane + 64u * j, row = H ? s / Y::SEGS : 4u * g + j / E, seg = H ? s % Y::SEGS : i + 16u * (j % E);
            vr[j] = *(const ju4 *)(at + (min(row, e1 - 1 - p) * kvrow + seg * 16u));
        }
    };
    uint32_t p = p0 + STEP * pg;
    if (p < e1) {
        load_k(p);
        load_v(p);
    }

    // q of the lane's columns
    constexpr int QN = D / 32;
    ph8 qh[H ? NT : 1][QN], ql[TWO ? NT : 1][QN];
    jf4 qf[H ? 1 : NT][D / 16];
    float sc2[NT], qs[NT];
    uint32_t lim[NT], qat[NT];
    const Q *qp[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const uint32_t c = min(c0 + 16u * n + i, ncols - 1), row = c / a.G;
        lim[n] = min(seen_of(w, row), p1);
        qat[n] = (w.row0 + row) * a.heads + kvh * a.G + (c - row * a.G);   // below 2^25
        qp[n] = (const Q *)a.q + (size_t)qat[n] * D;
        sc2[n] = a.scale2;
        qs[n] = 1.0f;
        if constexpr (!H) {
#pragma unroll
            for (int t = 0; t < D / 16; ++t) qf[n][t] = *(const jf4 *)(qp[n] + 16 * t + 4 * g);
        } else if constexpr (!TWO) {
#pragma unroll
            for (int t = 0; t < QN; ++t) qh[n][t] = *(const ph8 *)(qp[n] + 32 * t + 8 * g);
        } else {
            jf4 x[QN][2];
            float qmax = 0.0f;
#pragma unroll
            for (int t = 0; t < QN; ++t) {
                x[t][0] = *(const jf4 *)(qp[n] + 32 * t + 8 * g);
                x[t][1] = *(const jf4 *)(qp[n] + 32 * t + 8 * g + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) qmax = fmaxf(qmax, fmaxf(fabsf(x[t][0][e]), fabsf(x[t][1][e])));
            }
            qmax = fmaxf(qmax, swap16(qmax));
            qmax = fmaxf(qmax, swap32(qmax));
            const bool inf = qmax == INFINITY;
            qs[n] = inf ? 1.0f : two_part_scale(qmax);
            sc2[n] = a.scale2 / qs[n];
#pragma unroll
            for (int t = 0; t < QN; ++t)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float y = x[t][e >> 2][e & 3] * qs[n];
                    qh[n][t][e] = (_Float16)y;
                    ql[n][t][e] = (_Float16)(y - (float)qh[n][t][e]);
                }
            // beside an infinity of q no finite element counts, and it has one part
            if (__any(inf))
#pragma unroll
                for (int t = 0; t < QN; ++t)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float y = x[t][e >> 2][e & 3];
                        if (inf) {
                            qh[n][t][e] = (_Float16)(fabsf(y) == INFINITY ? y : y * 0.0f);
                            ql[n][t][e] = (_Float16)0.0f;
                        }
                    }
        }
    }
    const uint32_t lo = c0 < ncols ? min(seen_of(w, c0 / a.G), p1) : 0u;   // every column sees [0, lo)

    // q has arrived before the steps begin: a wait for it among them would be one for
    // the loads of the next step too
    if constexpr (!TWO) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int t = 0; t < (H ? QN : D / 16); ++t) {
                if constexpr (H) asm volatile("" : "+v"(qh[n][t]));
                else asm volatile("" : "+v"(qf[n][t]));
            }
    }
    pf4 o[NT][ND];
    float m[NT], l[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[n][d] = (pf4){};
    }
    unsigned char *vt = smem + wave * (32u * Y::RB);   // this wavefront's V tile (binary16)
    for (const uint32_t stride = pw * STEP; p < e1; p += stride) {
        const bool more = p + stride < e1;
        pf4 s[NT][NB];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                s[n][b] = (pf4){};
                pf4 s2 = (pf4){};
#pragma unroll
                for (int t = 0; t < KS; ++t) {
                    if constexpr (H) {
                        const ph8 k = __builtin_bit_cast(ph8, kr[b][t]);
                        s[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[n][t], s[n][b], 0, 0, 0);
                        if constexpr (TWO) s2 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[n][t], s2, 0, 0, 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float k = __uint_as_float(kr[b][t][e]);
                            if (t & 1) s2 = __builtin_amdgcn_mfma_f32_16x16x4f32(k, qf[n][t][e], s2, 0, 0, 0);
                            else s[n][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(k, qf[n][t][e], s[n][b], 0, 0, 0);
                        }
                    }
                }
                if constexpr (TWO || !H) {
#pragma unroll
                    for (int v = 0; v < 4; ++v) s[n][b][v] += s2[v];
                }
            }
        if constexpr (TWO) {
            float odd = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int t = 0; t < KS; ++t) odd = odd_sum<KV>(kr[b][t], odd);
            // an infinity of K times a part of q that is 0 or of the other sign would make a
            // NaN of an infinite score: such steps take q whole
            if (__any(odd != odd)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        s[n][b] = (pf4){};
#pragma unroll 1
                        for (int d = 0; d < D; d += 8) {
                            const jf4 q0 = *(const jf4 *)(qp[n] + d), q1 = *(const jf4 *)(qp[n] + d + 4);
#pragma unroll
                            for (int v = 0; v < 4; ++v) {
                                const uint32_t at = min(16u * b + 4u * g + v, e1 - 1 - p);
                                const ph8 k = *(const ph8 *)((const KV *)(kc + (size_t)(p + at) * kvrow) + d);
#pragma unroll
                                for (int e = 0; e < 8; ++e) s[n][b][v] = fmaf(e < 4 ? q0[e & 3] : q1[e & 3], (float)k[e], s[n][b][v]);
                            }
                        }
#pragma unroll
                        for (int v = 0; v < 4; ++v) s[n][b][v] *= qs[n];
                    }
            }
        }
        if (more) load_k(p + stride);
        // An infinity or NaN of V stays out of the products and is added on its own.
        float odd = 0.0f;
#pragma unroll
        for (int j = 0; j < VS; ++j) odd = odd_sum<KV>(vr[j], odd);
        uint32_t odd_v = 0;   // positions of the step that hold one
        if (__any(odd != odd)) {
#pragma unroll
            for (int j = 0; j < VS; ++j) {
                const float x = odd_sum<KV>(vr[j], 0.0f);
                const uint64_t hit = __ballot(x != x);
                constexpr uint32_t L = H ? Y::SEGS : 16;   // lanes of a position
#pragma unroll
                for (uint32_t r = 0; r < 64 / L; ++r)
                    if (hit >> (r * L) & ((1ull << L) - 1)) odd_v |= 1u << (H ? j * (64 / L) + r : 4 * r + j / (D / 64));
                vr[j] = finite_part<KV>(vr[j]);
            }
            if (e1 - p < STEP) odd_v &= (1u << (e1 - p)) - 1;   // behind the last position lie copies of it
        }
        if constexpr (H) {
#pragma unroll
            for (int j = 0; j < VS; ++j) {
                const uint32_t at = lane + 64u * j, row = at / Y::SEGS, seg = at % Y::SEGS;
                *(ju4 *)(vt + row * Y::RB + (seg ^ Y::few_swz(row)) * 16u) = vr[j];
            }
            if (more) load_v(p + stride);
        }
        if (p + STEP > lo) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int v = 0; v < 4; ++v) s[n][b][v] = p + 16 * b + 4 * g + v < lim[n] ? s[n][b][v] : -INFINITY;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float bm = -INFINITY;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int v = 0; v < 4; ++v) bm = fmaxf(bm, s[n][b][v]);
            bm = fmaxf(bm, swap16(bm));
            bm = fmaxf(bm, swap32(bm));
            if (__any((bm - m[n]) * sc2[n] > R::SLACK || (m[n] == -INFINITY && bm != -INFINITY))) {
                const float mn = fmaxf(m[n], bm), alpha = mn == m[n] ? 1.0f : __builtin_amdgcn_exp2f((m[n] - mn) * sc2[n]);
                m[n] = mn;
                l[n] *= alpha;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int v = 0; v < 4; ++v) o[n][d][v] *= alpha;
            }
            const float mr = m[n] == -INFINITY ? 0.0f : m[n];
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    s[n][b][v] = __builtin_amdgcn_exp2f(fmaf(s[n][b][v] - mr, sc2[n], R::BIAS));
                    sum += s[n][b][v];
                }
            l[n] += sum;
        }
        if constexpr (H) {
            ph8 ph[NT], pl[TWO ? NT : 1];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = s[n][e >> 2][e & 3];
                    ph[n][e] = (_Float16)x;
                    if constexpr (TWO) pl[n][e] = (_Float16)(x - (float)ph[n][e]);
                }
            // lane 16 g + i reads dims 16 d + 4 (i % 4) .. of position 4 g + i / 4 and
            // receives dim 16 d + i of positions 4 g .. 4 g + 3
            const uint32_t row = 4u * g + (i >> 2);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const uint32_t at = row * Y::RB + ((2u * d + ((i & 3u) >> 1)) ^ Y::few_swz(row)) * 16u + (i & 1u) * 8u;
                const ps4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(vt + at));
                const ps4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(vt + at + 16 * Y::RB));
                const ph8 v = __builtin_bit_cast(ph8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[n], o[n][d], 0, 0, 0);
                    if constexpr (TWO) o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[n], o[n][d], 0, 0, 0);
                }
            }
        } else {
            constexpr int E = D / 64;
#pragma unroll
            for (int v = 0; v < 4; ++v)
#pragma unroll
                for (int e = 0; e < E; ++e)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            o[n][4 * e + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[v * E + e][c]), s[n][0][v], o[n][4 * e + c], 0, 0, 0);
            if (more) load_v(p + stride);
        }
        if (odd_v) {
#pragma unroll 1
            for (; odd_v; odd_v &= odd_v - 1) {
                const uint32_t j = __builtin_ctz(odd_v);
                const KV *row = (const KV *)(vc + (size_t)(p + j) * kvrow);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float mine = 0.0f;
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int v = 0; v < 4; ++v) mine = 4u * (j >> 4) + (j & 3u) == 4u * b + v ? s[n][b][v] : mine;
                    const float pj = __int_as_float(__builtin_amdgcn_ds_bpermute((int)(((j >> 2) & 3u) * 16u + i) * 4, __float_as_int(mine)));
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            const float x = (float)row[H ? 16 * d + 4 * g + v : 4 * (4 * g + v + 16 * (d >> 2)) + (d & 3)];
                            if (p + j < lim[n] && (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) o[n][d][v] = fmaf(pj, x, o[n][d][v]);
                        }
                }
            }
        }
    }

    // join the wavefronts of a group
    const PackedArgs &z = late_args<PackedArgs>();
    constexpr uint32_t C = 16 * NT, OS = D + 4;    // padded: 16 columns meet 16 bank groups
    float *oo = (float *)smem;                     // [wave][column][OS], over the V tiles
    float2 *ml = (float2 *)(smem + 4 * C * OS * 4);   // [wave][column]
    float4 *fin = (float4 *)(ml + 4 * C);          // [group][column]: m, l, 1 / l, row and head
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        l[n] += swap16(l[n]);
        l[n] += swap32(l[n]);
        m[n] = m[n] / qs[n];
        if (g == 0) ml[wave * C + 16 * n + i] = make_float2(m[n], l[n]);
    }
    __syncthreads();   // also: every V tile has been read
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float2 all[4];   // of the group; a wavefront beyond it repeats one
        float M = -INFINITY, lt = 0.0f;
#pragma unroll
        for (uint32_t x = 0; x < 4; ++x) {
            all[x] = ml[(cg + min(x, pw - 1u) * cw) * C + 16 * n + i];
            M = fmaxf(M, all[x].x);
        }
#pragma unroll
        for (uint32_t x = 0; x < 4; ++x)
            if (x < pw) lt = fmaf(all[x].y, all[x].x == M ? 1.0f : __builtin_amdgcn_exp2f((all[x].x - M) * z.scale2), lt);
        const float f = m[n] == M ? 1.0f : __builtin_amdgcn_exp2f((m[n] - M) * z.scale2);
        float *to = oo + (wave * C + 16 * n + i) * OS;
        if constexpr (H) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
                *(jf4 *)(to + 16 * d + 4 * g) = jf4{o[n][d][0] * f, o[n][d][1] * f, o[n][d][2] * f, o[n][d][3] * f};
        } else {
#pragma unroll
            for (int e = 0; e < D / 64; ++e)
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    *(jf4 *)(to + 4 * (4 * g + v + 16 * e)) = jf4{o[n][4 * e][v] * f, o[n][4 * e + 1][v] * f, o[n][4 * e + 2][v] * f, o[n][4 * e + 3][v] * f};
        }
        if (pg == 0 && g == 0)   // a row that sees nothing is 0
            fin[cg * C + 16 * n + i] = make_float4(M, lt, lt == 0.0f ? 0.0f : 1.0f / lt, __uint_as_float(qat[n]));
    }
    __syncthreads();
    const uint32_t cols = min(C * cw, ncols - w.c0);
    for (uint32_t at = tid; at < cols * (D / 4); at += 256) {
        const uint32_t x = at / (D / 4), dim = at % (D / 4) * 4u, group = x / C;
        const float4 f = fin[x];
        const float *from = oo + (size_t)(group * C + x % C) * OS + dim;   // wavefront `group`, then every cw-th
        jf4 sum = *(const jf4 *)from;
        for (uint32_t y = 1; y < pw; ++y) {
            const jf4 more = *(const jf4 *)(from + y * cw * C * OS);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += more[e];
        }
        const size_t to = __float_as_uint(f.w);
        if (z.slots) {
            const size_t part = to * z.slots + w.slot;
            if (dim == 0) *(float2 *)(z.part_ml + 2 * part) = make_float2(f.x, f.y);
            *(jf4 *)(z.part + part * D + dim) = sum;
        } else {
            typedef Q q4 __attribute__((ext_vector_type(4)));
            q4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (Q)(sum[e] * f.z);
            *(q4 *)((Q *)z.out + to * D + dim) = y;
        }
    }
}

// Up to 128 columns on a binary16 cache: K and V pass through LDS for all four
// wavefronts, 32 columns each, requested a tile of TP positions ahead straight into LDS.
//
// The vector unit is as busy as the matrix unit (a wavefront's tile of 64 positions
// is 32 MFMAs of 17 ns, about 100 other instructions of 2.1 ns and 32 exponentials
// of 5.2 ns, and only the exponentials overlap with the MFMAs of the other
// wavefront in full), so whatever a score does not need is kept out: no look at the
// values on their way (an infinity or NaN shows in the sums at the end, and the
// wavefront then takes odd_columns), offsets made once, l summed from pairs of P.
// Tried and slower: the scores of the next tile before the softmax of this one
// (32 registers more, which spill).
//   S^T: position 8 (v / 4) + 4 h + v % 4 of column lane % 32 in s[v], h = lane / 32
template <typename Q, int D, int TP>
__device__ __forceinline__ bool wide_tile(const PackedArgs &a, const Work &w, uint32_t kvh, uint32_t ncols, uint32_t p0,
                                          uint32_t p1, unsigned char *smem) {
    typedef Range<Q, _Float16> R;
    typedef Lay<D> Y;
    constexpr bool TWO = R::TWO;
    constexpr int NB = TP / 32, ND = D / 32, QN = D / 16;
    constexpr uint32_t TB = TP * Y::RB;            // bytes of a tile of K or V; LDS: K, V, K, V
    constexpr int LD = TB / 4096;                  // 1 KB requests per wavefront and tile
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t col = lane & 31u, h = lane >> 5;
    const uint32_t kvrow = a.kv_heads * Y::RB;     // bytes from a position to the next
    const unsigned char *kc = (const unsigned char *)a.kc + (w.kv_row * a.kv_heads + kvh) * Y::RB;
    const unsigned char *vc = (const unsigned char *)a.vc + (w.kv_row * a.kv_heads + kvh) * Y::RB;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)smem;
    // request j of this wavefront: row and permuted segment of its lanes
    auto row_of = [&](int j) { return (lane + 64u * (wave * LD + j)) / Y::SEGS; };
    auto seg_of = [&](int j, bool v) { return (lane % Y::SEGS ^ (v ? Y::v_swz(row_of(j)) : Y::k_swz(row_of(j)))) * 16u; };
    uint32_t ko[LD], vo[LD];
#pragma unroll
    for (int j = 0; j < LD; ++j) {
        ko[j] = row_of(j) * kvrow + seg_of(j, false);
        vo[j] = row_of(j) * kvrow + seg_of(j, true);
    }
    // the tile of positions from p on into buffer b: K, then V
    auto request = [&](uint32_t p, uint32_t b) {
        const unsigned char *kp = kc + (size_t)p * kvrow, *vp = vc + (size_t)p * kvrow;
        const uint32_t to = lds0 + b * 2 * TB + wave * LD * 1024u;
        if (p + TP <= p1) {
#pragma unroll
            for (int j = 0; j < LD; ++j) {
                lds_request<false>(kp, ko[j], to + j * 1024u);
                lds_request<false>(vp, vo[j], to + TB + j * 1024u);
            }
        } else {   // rows beyond the part repeat its last one
#pragma unroll
            for (int j = 0; j < LD; ++j) {
                const uint32_t at = min(row_of(j), p1 - 1 - p) * kvrow;
                lds_request<false>(kp, at + seg_of(j, false), to + j * 1024u);
                lds_request<false>(vp, at + seg_of(j, true), to + TB + j * 1024u);
            }
        }
    };
    uint32_t *again = (uint32_t *)(smem + 4 * TB);   // behind the tiles
    if (threadIdx.x == 0) *again = 0;
    if (p0 < p1) request(p0, 0);

    const uint32_t wc0 = w.c0 + 32u * wave;
    const bool idle = wc0 >= ncols;     // uniform: this wavefront only helps to load
    const uint32_t wave_lo = idle ? 0u : seen_of(w, wc0 / a.G);
    const uint32_t wave_hi = idle ? 0u : min(seen_of(w, min(wc0 + 31u, ncols - 1) / a.G), p1);
    const uint32_t c = min(wc0 + col, ncols - 1), qrow = c / a.G, head = kvh * a.G + (c - qrow * a.G);
    const uint32_t lim = min(seen_of(w, qrow), p1);
    const size_t qat = ((size_t)(w.row0 + qrow) * a.heads + head);

    // q of this lane's column
    const Q *qp = (const Q *)a.q + qat * D;
    ph8 qh[QN], ql[TWO ? QN : 1];
    float sc2 = a.scale2, qs = 1.0f;
    if constexpr (!TWO) {
#pragma unroll
        for (int s = 0; s < QN; ++s) qh[s] = *(const ph8 *)(qp + 16 * s + 8 * h);
    } else {
        float qmax = 0.0f;
        jf4 x[QN][2];
#pragma unroll
        for (int s = 0; s < QN; ++s) {
            x[s][0] = *(const jf4 *)(qp + 16 * s + 8 * h);
            x[s][1] = *(const jf4 *)(qp + 16 * s + 8 * h + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) qmax = fmaxf(qmax, fmaxf(fabsf(x[s][0][i]), fabsf(x[s][1][i])));
        }
        qs = two_part_scale(fmaxf(qmax, swap32(qmax)));
        sc2 /= qs;
#pragma unroll
        for (int s = 0; s < QN; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = x[s][i >> 2][i & 3] * qs;
                qh[s][i] = (_Float16)y;
                ql[s][i] = (_Float16)(y - (float)qh[s][i]);
            }
    }

    pf16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = (pf16){};
    // p = 2^(s sc2 + c), c = BIAS - m sc2 rounded: one FMA a score
    float m = -INFINITY, c2 = INFINITY, l = 0.0f;
    // q has arrived before the tiles begin: the compiler's wait for it among them
    // would be one for the next tile too
    if constexpr (!TWO) {
#pragma unroll
        for (int t = 0; t < QN; ++t) asm volatile("" : "+v"(qh[t]));
    }
    // lanes 16 g + i of half h read dims 32 d + 16 g + 4 (i % 4) .. of positions
    // 4 h + i / 4 (+ 8) of a step of V and receive dim 32 d + 16 g + i of four positions
    const uint32_t vrow = 4u * h + ((lane & 15u) >> 2);
    const uint32_t vat = vrow * Y::RB + ((2u * ((lane >> 4) & 1u) + ((lane & 3u) >> 1)) ^ Y::v_swz(vrow)) * 16u + (lane & 1u) * 8u;
    const uint32_t kat = col * Y::RB + (h ^ Y::k_swz(col)) * 16u;
    uint32_t b = 0;
    for (uint32_t p = p0; p < p1; p += TP, b ^= 1u) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();   // this tile is there, the other buffer has been read
        if (p + TP < p1) request(p + TP, b ^ 1u);
        if (p >= wave_hi) continue;
        const unsigned char *kt = smem + b * 2 * TB, *vt = kt + TB;
        pf16 s[NB];
        ph8 k[NB][QN];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int t = 0; t < QN; ++t) k[n][t] = *(const ph8 *)(kt + (kat ^ (t * 32u)) + n * 32 * Y::RB);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            s[n] = (pf16){};
            if constexpr (TWO)   // the small parts first
#pragma unroll
                for (int t = 0; t < QN; ++t) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[n][t], ql[t], s[n], 0, 0, 0);
#pragma unroll
            for (int t = 0; t < QN; ++t) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[n][t], qh[t], s[n], 0, 0, 0);
        }
        // The operands of 32 positions (of half their dims in tiles of 32, which saves
        // registers) are requested together, and the next ones one by one behind the
        // products: left to itself the compiler waits for each before it asks for the next.
        constexpr int AHEAD = NB == 2 || TWO ? QN : QN / 2;
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
        if constexpr (!TWO)
#pragma unroll
            for (int t = 0; t < NB * QN - AHEAD; ++t) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
        __builtin_amdgcn_sched_group_barrier(0x008, TWO ? 2 * QN : AHEAD, 0);
        if (p + TP > min(wave_lo, p1)) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int v = 0; v < 16; ++v) s[n][v] = p + 32 * n + 8 * (v >> 2) + 4 * h + (v & 3) < lim ? s[n][v] : -INFINITY;
        }
        float top[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            top[v] = s[0][v];
#pragma unroll
            for (int x = v + 2; x < 16 * NB; x += 2) top[v] = fmaxf(top[v], s[x >> 4][x & 15]);
        }
        float bm = fmaxf(top[0], top[1]);
        bm = fmaxf(bm, swap32(bm));
        if (__any(fmaf(bm, sc2, c2) > R::BIAS + R::SLACK)) {
            m = fmaxf(m, bm);
            const float cn = fmaf(-m, sc2, R::BIAS), alpha = cn == c2 ? 1.0f : __builtin_amdgcn_exp2f(cn - c2);
            c2 = cn;
            l *= alpha;
            // scores so large that c does not hold their last bits: few_columns takes the difference instead
            if (fabsf(c2) > 4194304.0f && m != -INFINITY) l = NAN;   // c itself may be infinite
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[d][v] *= alpha;
        }
        // while only masked or NaN scores have come, m counts as 0: 2^-inf is 0, a NaN stays
        const float c0 = c2 == INFINITY ? 0.0f : c2;
        float sum[2] = {};
#pragma unroll
        for (int t = 0; t < 2 * NB; ++t) {
            ph8 ph, pl;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = s[t >> 1][8 * (t & 1) + e];
                const float x = __builtin_amdgcn_exp2f(fmaf(y, sc2, c0));
                ph[e] = (_Float16)x;
                if constexpr (TWO) {
                    pl[e] = (_Float16)fmaf((float)ph[e], -1.0f, x);
                    sum[e & 1] += x;
                }
            }
            if constexpr (!TWO) {   // of P as rounded: both sums see the same weights
                const jh2 one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
                for (int e = 0; e < 8; e += 2) sum[(e >> 1) & 1] = __builtin_amdgcn_fdot2(jh2{ph[e], ph[e + 1]}, one, sum[(e >> 1) & 1], false);
            }
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const unsigned char *at = vt + (vat ^ (d * 64u)) + 16 * t * Y::RB;
                const ps4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)at);
                const ps4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(at + 8 * Y::RB));
                const ph8 v = __builtin_bit_cast(ph8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph, o[d], 0, 0, 0);
                if constexpr (TWO) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl, o[d], 0, 0, 0);
            }
        }
        l += sum[0] + sum[1];
    }

    l += swap32(l);
    // an infinity or NaN anywhere makes the sum a NaN
    float odd = l * 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) odd = fmaf(o[d][v], 0.0f, odd);
    if (p0 < p1) {   // else nothing is odd, and no barrier has followed the 0
        if (__any(odd != odd) && lane == 0) *again = 1;
        __syncthreads();
        if (__builtin_amdgcn_readfirstlane(*again)) return true;
    }
    if (wc0 + col >= ncols) return false;
    const PackedArgs &z = late_args<PackedArgs>();
    if (z.slots) {
        const size_t at = qat * z.slots + w.slot;
        // what the rounding of c shifted, since the parts are joined by m
        const float back = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(R::BIAS - fmaf(m, sc2, c2));
        if (h == 0) *(float2 *)(z.part_ml + 2 * at) = make_float2(m / qs, l * back);
        if (p0 >= p1) return false;   // the join reads no output of a part without positions
        float *to = z.part + at * D;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *(jf4 *)(to + 32 * d + 8 * j + 4 * h) = jf4{o[d][4 * j] * back, o[d][4 * j + 1] * back, o[d][4 * j + 2] * back, o[d][4 * j + 3] * back};
        return false;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;   // a row that sees nothing is 0
    Q *to = (Q *)z.out + qat * D;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            typedef Q q4 __attribute__((ext_vector_type(4)));
            q4 y;
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = (Q)(o[d][4 * j + i] * inv);
            *(q4 *)(to + 32 * d + 8 * j + 4 * h) = y;
        }
    return false;
}

// Kernels of a launch. Few: 16 columns per workgroup, whose LDS and registers let three
// workgroups share a CU (with 128 dims and two parts two: three would spill, and scratch
// costs half the rate; with 64 dims four). 24 sequences of 2 to 50 rows behind up to 200
// at 16/1/128, binary32: 25.1 us with two, 22.7 with three. Light (binary16 rows, 128
// dims): all columns through wide_tile in tiles of 32 positions, three workgroups on a
// CU too. Any: the others.
enum Kind { Any, Few, Light };
template <typename Q, typename KV, int D, Kind K> constexpr int per_cu() {
    if (D == 128) return K == Any || Range<Q, KV>::TWO ? 2 : 3;
    return K == Few ? 4 : 2;
}

// Q: _Float16 or float rows; KV: the cache's type.
template <typename Q, typename KV, int D, Kind K>
__global__ __launch_bounds__(256, (per_cu<Q, KV, D, K>())) void packed_attn_kernel(PackedArgs a) {
    constexpr bool H = sizeof(KV) == 2;
    extern __shared__ __align__(16) unsigned char smem[];
    // Neighbouring workgroups take the KV heads, so that with 8 of them each XCD keeps
    // the K and V of one head in its L2. The prefix's workgroups come first: every CU
    // gets one, then those of the requests' own positions.
    const bool shared = blockIdx.x < a.prefix_blocks;
    const uint32_t block = blockIdx.x - (shared ? 0u : a.prefix_blocks);
    const uint32_t kvh = block % a.kv_heads, id = block / a.kv_heads;
    Work w;
    if (shared) {
        w.part = id % a.prefix_splits;
        w.parts = a.prefix_splits;
        w.chunk = ((a.prefix_len + a.prefix_splits - 1) / a.prefix_splits + 63u) / 64u * 64u;
        w.slot = w.part;
        w.row0 = 0;
        w.n = a.rows;
        w.c0 = id / a.prefix_splits * a.cols;
        w.kv_row = a.prefix_row;
        w.len = a.prefix_len;
        w.first = 0;
        w.causal = false;
    } else {
        if (!find_task(a, id, w)) return;
        w.slot = a.prefix_splits + w.part;
    }
    const uint32_t ncols = min(w.n * a.G, w.c0 + a.cols);   // up to the tile's last column; n G < 2^25
    const uint32_t end_all = seen_of(w, (ncols - 1) / a.G);
    const uint32_t p0 = min(w.part * w.chunk, end_all), p1 = min(p0 + w.chunk, end_all);
    if (!shared && a.slots && w.part + 1 == w.parts && w.parts < a.splits) {   // parts that there are none of
        const uint32_t none = a.splits - w.parts, cols = ncols - w.c0;
        for (uint32_t x = threadIdx.x; x < cols * none; x += 256) {
            const uint32_t c = w.c0 + x / none, row = c / a.G;
            const size_t qat = (size_t)(w.row0 + row) * a.heads + kvh * a.G + (c - row * a.G);
            *(float2 *)(a.part_ml + 2 * (qat * a.slots + w.slot + 1 + x % none)) = make_float2(-INFINITY, 0.0f);
        }
    }
    if constexpr (K == Few) {
        few_columns<Q, KV, D, 1>(a, w, kvh, ncols, p0, p1, 1, smem);
        return;
    }
    const uint32_t cols = ncols - w.c0;
    bool wide = H, again = false;
    if constexpr (K == Light) again = wide_tile<Q, D, 32>(a, w, kvh, ncols, p0, p1, smem);
    if constexpr (H && K == Any) {
        // Few columns of a split context on binary16 rows: one wavefront computes and all
        // four request, a tile of 32 positions ahead, which keeps more reads in flight than
        // few_columns does (five tokens each of 16 requests behind up to 4000 positions: 33
        // us against 36; one each: 36 either way). Not worth its start where parts are short
        // and columns few or nothing is split (five tokens of one request behind 600: 16.0
        // against 12.4, of 16 behind up to 600: 16.3 against 13.6), nor with the products of
        // two parts.
        const bool narrow = sizeof(Q) == 2 && (shared ? cols > 16 : a.splits > 1 && (cols > 16 || w.chunk >= 256));
        if (cols > few_of<Q, KV>()) again = wide_tile<Q, D, sizeof(Q) == 2 ? 64 : 32>(a, w, kvh, ncols, p0, p1, smem);
        else if (narrow) again = wide_tile<Q, D, 32>(a, w, kvh, ncols, p0, p1, smem);
        else wide = false;
    }
    if (wide && !__builtin_amdgcn_readfirstlane(again)) return;   // one value for the workgroup
    if constexpr (few_of<Q, KV>() == 32 && K == Any) {
        if (!wide && cols > 16) {
            few_columns<Q, KV, D, 2>(a, w, kvh, ncols, p0, p1, cols > 32 ? 2 : 1, smem);
            return;
        }
    }
    // 16 columns, or all of a tile that met an infinity, a NaN or a score beyond 2^22. One
    // prompt of 2048 rows at 32/8/128 with such a value at position 0, which every tile
    // sees: 290 us, 56 without (binary16); 415 and 92 (two parts).
    for (;;) {
        few_columns<Q, KV, D, 1>(late_args<PackedArgs>(), w, kvh, ncols, p0, p1, 1, smem);
        if ((w.c0 += 16) >= ncols) return;
        __syncthreads();   // the outputs have been read from LDS
    }
}

// Joins the parts of a row and head: a wavefront each. A part holds m, l and the
// output before the division; one without positions has l = 0 and no output, one
// with only NaN scores an m of -infinity and a NaN l.
template <typename Q, int D>
__global__ __launch_bounds__(256) void packed_join_kernel(PackedArgs a) {
    const uint64_t at = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63u, row = (uint32_t)(at / a.heads);
    if (row >= a.rows) return;
    // rows outside the sequences are not written
    if (a.q_start && ((int32_t)row < a.q_start[0] || (int32_t)row >= a.q_start[a.nseq])) return;
    constexpr int E = D / 64;
    const float2 *ml = (const float2 *)a.part_ml + at * a.slots;
    const float *part = a.part + at * a.slots * D + E * lane;
    constexpr int U = 8;
    typedef float vec __attribute__((ext_vector_type(E)));
    float M = -INFINITY, l = 0.0f;
    vec o = {};
    for (uint32_t s0 = 0; s0 < a.slots; s0 += 64) {   // lane s: part s0 + s
        const float2 p = s0 + lane < a.slots ? ml[s0 + lane] : make_float2(-INFINITY, 0.0f);
        const float m0 = M;
        M = fmaxf(M, wave_max(p.x));
        const float w = p.y == 0.0f ? 0.0f : p.x == M ? 1.0f : __builtin_amdgcn_exp2f((p.x - M) * a.scale2);
        const float old = M == m0 ? 1.0f : __builtin_amdgcn_exp2f((m0 - M) * a.scale2);
        l = fmaf(l, old, wave_sum(p.y * w));
        o *= old;
        // U parts in flight; those without positions repeat the first that has some
        const uint64_t has = __ballot(p.y != 0.0f);
        if (!has) continue;
        const uint32_t first = __ffsll((unsigned long long)has) - 1, n = 64 - __builtin_clzll(has);
        for (uint32_t s = 0; s < n; s += U) {
            vec x[U];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const uint32_t k = s + u < 64 && (has >> ((s + u) & 63) & 1) ? s + u : first;
                x[u] = *(const vec *)(part + (size_t)(s0 + k) * D);
            }
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const bool there = s + u < 64 && (has >> ((s + u) & 63) & 1);
                const float wu = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), (s + u) & 63));
#pragma unroll
                for (int i = 0; i < E; ++i) o[i] = there ? fmaf(x[u][i], wu, o[i]) : o[i];
            }
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < E; ++i) ((Q *)a.out)[at * D + E * lane + i] = (Q)(o[i] * inv);
}

template <typename Q, typename KV, int D, Kind K>
int launch_attn(janus_ctx *ctx, const PackedArgs &a, uint32_t blocks) {
    // two tiles of K and V (a V tile per wavefront) and a flag, or the join of the wavefronts of few columns
    constexpr size_t tiles = sizeof(KV) == 2 ? 4 * (sizeof(Q) == 2 && K == Any ? 64 : 32) * D * 2 + 16 : 0;
    constexpr size_t held = K == Any ? 32 : 16;
    constexpr size_t lds = std::max<size_t>(tiles, 4 * held * ((D + 4) * 4 + 8) + 2 * held * 16);
    static std::atomic<uint64_t> asked{0};   // devices on which the kernel may take that much
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (!(asked.load(std::memory_order_relaxed) & bit)) {
        JANUS_HIP_CHECK(ctx, hipFuncSetAttribute((const void *)packed_attn_kernel<Q, KV, D, K>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, lds));
        asked.fetch_or(bit, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL((packed_attn_kernel<Q, KV, D, K>), dim3(blocks), dim3(256), lds, ctx->stream, a);
    JANUS_LAUNCH_CHECK(ctx);
    return JANUS_OK;
}

template <typename Q, typename KV, int D>
int launch(janus_ctx *ctx, const PackedArgs &a, uint32_t blocks) {
    int e = JANUS_OK;
    if (a.cols == 16) {
        e = launch_attn<Q, KV, D, Few>(ctx, a, blocks);
    } else if (a.light) {
        if constexpr (sizeof(Q) == 2 && D == 128) e = launch_attn<Q, KV, D, Light>(ctx, a, blocks);
    } else {
        e = launch_attn<Q, KV, D, Any>(ctx, a, blocks);
    }
    if (e) return e;
    if (a.slots) {
        const uint64_t heads = (uint64_t)a.rows * a.heads;
        hipLaunchKernelGGL((packed_join_kernel<Q, D>), dim3((uint32_t)((heads + 3) / 4)), dim3(256), 0, ctx->stream, a);
        JANUS_LAUNCH_CHECK(ctx);
    }
    return JANUS_OK;
}

int launch_typed(janus_ctx *ctx, const PackedArgs &a, int q_dt, int kv_dt, uint32_t hd, uint32_t blocks) {
    if (q_dt == JANUS_DT_F16) return hd == 64 ? launch<_Float16, _Float16, 64>(ctx, a, blocks) : launch<_Float16, _Float16, 128>(ctx, a, blocks);
    if (kv_dt == JANUS_DT_F16) return hd == 64 ? launch<float, _Float16, 64>(ctx, a, blocks) : launch<float, _Float16, 128>(ctx, a, blocks);
    return hd == 64 ? launch<float, float, 64>(ctx, a, blocks) : launch<float, float, 128>(ctx, a, blocks);
}

// Parts of a tile so that `tiles` of them fill the CUs (two workgroups on each),
// each with `least` positions at least.
uint32_t plan_splits(const janus_ctx *ctx, uint64_t tiles, uint32_t max_len, uint32_t least) {
    const uint64_t want = 2ull * ctx->num_cus / std::max<uint64_t>(tiles, 1);
    return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(want, (max_len + least - 1) / least));
}

// Whether q and P are in two parts (binary32 rows on a binary16 cache).
bool two_parts(int q_dt, int kv_dt) { return q_dt != kv_dt; }

// The parts of a request's own positions, where `likely` tiles are expected and
// there are at most `tiles`: returns the tasks per KV head. Parts cost a second
// launch (about 5 us) unless the results are joined anyway, and where there is a tile
// for nearly every CU a second workgroup on each gains only a quarter to a third. So
// contexts stay whole below some lengths, by the time that a position takes (one
// prompt of 512 rows at 32/8/128 in binary16: 15 us in one part, 22 in two).
uint64_t plan_own(const janus_ctx *ctx, PackedArgs &a, int q_dt, int kv_dt, uint64_t columns, uint64_t likely,
                  uint64_t tiles, uint32_t max_len) {
    const bool cheap = q_dt == JANUS_DT_F16 || (two_parts(q_dt, kv_dt) && a.cols == 16);
    const bool busy = 3 * likely * a.kv_heads >= 2ull * (uint32_t)ctx->num_cus;
    const uint32_t whole = a.prefix_splits ? 0 : cheap ? (busy ? 1280 : 640) : busy ? 768 : 384;
    // parts of 256 positions, where more than 16 columns go through LDS (four tiles of 64)
    const uint32_t least = q_dt == JANUS_DT_F16 && columns > 16 && a.cols > 32 && !a.prefix_splits ? 256 : 128;
    const uint32_t want = max_len < whole ? 1 : plan_splits(ctx, likely * a.kv_heads, max_len, least);
    a.splits = 1;
    if (want == 1) return tiles;
    // of several requests one may take four times the mean (the workspace is sized for that)
    a.splits = a.nseq == 1 ? want : std::min(4 * want, std::max(2u, (max_len + 127) / 128));
    a.target = std::max(1u, 2u * (uint32_t)ctx->num_cus / a.kv_heads);
    return tiles + a.target + 1;   // sum of tiles * ceil(len / chunk) <= target + tiles
}

// Columns per workgroup for `groups` runs of `columns` columns each on up to max_len
// positions (of the caches' capacity, where the caller gave no hint). Many columns
// share the K and V that a workgroup reads and few fill the CUs without splitting the
// positions. Us with 128, 64, 32 and 16 (binary32 caches: 64, 32, 16), * what is taken,
// at 32/8/128 unless named; requests behind a prefix have up to 40 positions of their own:
//                               binary16              two parts             binary32
//   one prompt of 256           11.1 9.9 10.0 9.9*    16.5 15.2 14.2 11.9*  26.8 17.9 15.2*
//   one prompt of 1024          26* 26 36 47          54* 40 46 58          110 97* 99
//     at 24/8/64                17* 17 17 23          34* 27 26 26          58 44* 48
//   11 prompts of 12 to 244     17.7* 17.7 32 33      25* 28 37 50          48* 60 58
//     at 40/8/128               19* 21 39 40          28* 32 44 62          59* 76 74
//   30 rows behind 500          16 15 12.6 10.3*      16 15 13.7 11.6*      22 17 16*
//   3 of 2 to 40 behind 900     14.1 12.5 13.5 14.6*  17 15 16 19*          23 24 21*
//     behind 1900               15.6* 15.8 15.2 18    19* 19 18 22          28 26 29*
//   16 times 5 rows behind 400  12.1 12.2 12.2 10.1*  16 16 16 11.5*        24 24 17*
//     behind 1000               19* 19 19 15          24 24 24 16*          35* 35 30
//     behind 1200               15* 15 15 17          20 19 19 18*          31* 31 34
//     behind 4000               43* 43 43 51          50* 50 50 53          80 80* 92
//   16 times 12 behind 4000     47* 47 60 73          55* 55 76 75          129* 123 153
//   16 requests, prefix of 500  10.6 10.7* 10.3 10.5  13 13 13 10.2*        20 15 11*
//   22 of 500                   11.7 10.9* 10.5 10.0  15 13 13 11.6*        20 16 13*
//   8 of 10000                  16.6 16.6 16.7 16.3*  21 21 21 17*          29 28 28*
//   22 of 10000                 19* 22 28 27          25* 31 39 28          62 52* 60
//   64 of 4000                  20* 20 28 28          25* 27 39 30          54 52* 57
//   45 of 2000 at 32/32/128     20.0 20.0 24 19.9*    29 29 28 27*          43 39* 38
//   32 of 4096 at 40/8/128      19* 19 23 23          24* 26 31 25          48 41* 44
//     at 24/8/64                13* 13 15 13          15.3 16 18 14.4*      23 21* 21
// Once a context is long enough to be split, the columns of a sequence stay together,
// since each tile of them reads K and V.
uint32_t plan_cols(const janus_ctx *ctx, const PackedArgs &a, int q_dt, int kv_dt, uint64_t groups, uint64_t columns,
                   uint32_t max_len) {
    const uint64_t cus = (uint64_t)ctx->num_cus, load = columns * a.kv_heads;
    auto tiles = [&](uint32_t cols) { return groups * ((columns + cols - 1) / cols) * a.kv_heads; };
    if (kv_dt != JANUS_DT_F16) {
        if (a.prefix_len) {
            if (load >= 32 * cus) return 64;
            return a.prefix_len >= 1024 && load >= (a.prefix_len >= 4096 ? 2 : 4) * cus ? 32 : 16;
        }
        if (columns > 16 && columns <= 32 && max_len > 550) return 32;
        if (columns > 32 && columns <= 64 && max_len > 1100) return 64;
        if (tiles(64) >= (max_len <= 128 ? cus * 3 / 4 : max_len <= 256 ? cus * 7 / 4 : 3 * cus)) return 64;
        return max_len > 256 && tiles(32) >= 2 * cus ? 32 : 16;
    }
    const bool two = two_parts(q_dt, kv_dt);
    if (!a.prefix_len && columns > 32 && max_len <= 1100 && tiles(16) <= (two && max_len > 512 ? 3 : 2) * cus) return 16;
    if (two) {
        if (columns <= 16 || (columns <= 32 && max_len <= 1200)) return 16;
        if (a.prefix_len) {
            if (load <= 6 * cus && load * max_len <= 16384 * cus) return 16;
        } else if (max_len <= 512 && tiles(16) <= (max_len <= 256 ? 2 : 4) * cus) {
            return 16;
        }
    }
    if (a.prefix_len && !two) {   // long ones, or many requests' own positions beside the prefix's
        if (max_len >= 4096 && load * max_len <= 10400 * cus) return 16;
        if ((uint64_t)a.rows * a.kv_heads >= 2 * cus && load * max_len <= 12288 * cus) return 16;
    }
    if (tiles(128) >= cus * 3 / 4) return 128;
    return max_len <= (a.prefix_len && !two ? 2048 : 1024) ? 64 : 128;
}

int run(janus_ctx *ctx, PackedArgs a, int q_dt, int kv_dt, uint32_t hd, uint64_t own_tasks) {
    const uint64_t prefix = (uint64_t)a.prefix_tiles * a.prefix_splits * a.kv_heads, own = own_tasks * a.kv_heads;
    // with rows * heads below 2^25 only where sequences * kv_heads is 2^23 or more
    if ((prefix + own) * 256 >= (1ull << 32))
        return fail(ctx, JANUS_E_INVALID_DIM, "attention: more sequences than one launch takes");
    a.prefix_blocks = (uint32_t)prefix;
    if (a.slots) {
        const size_t parts = (size_t)a.rows * a.heads * a.slots;
        if (int e = ensure_attn_ws(ctx, parts * (hd + 2) * sizeof(float))) return e;
        a.part = (float *)ctx->attn_ws;
        a.part_ml = a.part + parts * hd;
    }
    return launch_typed(ctx, a, q_dt, kv_dt, hd, (uint32_t)(prefix + own));
}

}  // namespace

int prompt_attention_launch(janus_ctx *ctx, const void *q, int q_dt, const void *kc, const void *vc, int kv_dt,
                            void *out, uint32_t rows, uint32_t nseq, uint32_t heads, uint32_t kv_heads, uint32_t hd,
                            uint32_t max_seq, const int32_t *q_start, const int32_t *row_base,
                            const int32_t *seq_lens, uint32_t max_len, float scale) {
    PackedArgs a{};
    a.q = q; a.kc = kc; a.vc = vc; a.out = out;
    a.q_start = q_start; a.row_base = row_base; a.seq_lens = seq_lens;
    a.rows = rows; a.nseq = nseq; a.heads = heads; a.kv_heads = kv_heads; a.G = heads / kv_heads;
    a.max_seq = max_seq;
    a.seq_len = -1;
    a.scale2 = scale * 1.4426950408889634f;
    max_len = std::min({max_len, max_seq, 0x7fffffffu});
    if (!seq_lens) max_len = std::min(max_len, q_start ? rows : rows / nseq);
    const uint64_t mean = (uint64_t)((rows + nseq - 1) / nseq) * a.G;   // columns of a sequence
    const uint32_t cols = a.cols = plan_cols(ctx, a, q_dt, kv_dt, nseq, mean, max_len);
    // at most so many tiles: every sequence's last one may be part empty
    const uint64_t tiles = (uint64_t)rows * a.G / cols + nseq;
    // about as many as sequences of equal rows have
    const uint64_t likely = (uint64_t)nseq * ((mean + cols - 1) / cols);
    const uint64_t tasks = plan_own(ctx, a, q_dt, kv_dt, mean, likely, tiles, max_len);
    a.slots = a.splits > 1 ? a.splits : 0;
    // Three light workgroups hide each other's start, where there are more than two for
    // each CU, on long contexts three (24 prompts of 3 to 700 rows: 70 us against 75; one
    // of 8192: 557 against 560; 24 of 7 to 150 behind up to 600: 36 against 35; three of 45
    // to 900, 576 workgroups: 32.2 against 31.4).
    a.light = q_dt == JANUS_DT_F16 && hd == 128 && cols >= 64 && a.splits == 1 &&
              likely * kv_heads > (max_len <= 800 ? 2u : 3u) * (uint32_t)ctx->num_cus;
    a.longest = kv_dt != JANUS_DT_F16 && a.splits == 1 && nseq > 1 && nseq <= 64 && likely * kv_heads > 2u * (uint32_t)ctx->num_cus;
    return run(ctx, a, q_dt, kv_dt, hd, tasks);
}

int prefix_attention_launch(janus_ctx *ctx, const void *q, int q_dt, const void *kc, const void *vc, int kv_dt,
                            void *out, uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t hd,
                            uint32_t prefix_row, uint32_t prefix_len, uint32_t seq_len, uint32_t max_seq,
                            const int32_t *row_base, const int32_t *seq_lens, uint32_t max_len, float scale) {
    PackedArgs a{};
    a.q = q; a.kc = kc; a.vc = vc; a.out = out;
    a.row_base = row_base; a.seq_lens = seq_lens;
    a.rows = a.nseq = batch; a.heads = heads; a.kv_heads = kv_heads; a.G = heads / kv_heads;
    a.max_seq = max_seq;
    a.seq_len = seq_len;
    a.prefix_row = prefix_row; a.prefix_len = prefix_len;
    a.scale2 = scale * 1.4426950408889634f;
    max_len = std::min({max_len, max_seq, 0x7fffffffu});
    const uint32_t cols = a.cols = plan_cols(ctx, a, q_dt, kv_dt, 1, (uint64_t)batch * a.G, std::max(prefix_len, max_len));
    const uint64_t own_tiles = (uint64_t)batch * ((a.G + cols - 1) / cols);
    if (prefix_len) {
        a.prefix_tiles = (uint32_t)(((uint64_t)batch * a.G + cols - 1) / cols);
        // At most one workgroup per CU, beside those of the own positions: half the
        // partials of two per CU (64 requests behind 16384 positions: 61 against 69 us, in
        // two parts 67 against 85; 32 behind 8192 with one own: 20 either way). A part
        // reads K and V once and writes a row per column, so it has at least two positions
        // for each column, and 128 for the four wavefronts (16 requests behind 3000
        // positions: 12.5 us, with 256 13.1, with 512 17; 32 behind 4096: 16.3 us with 256,
        // 17.3 with 128, 19 with 512).
        const uint32_t held = (uint32_t)std::min<uint64_t>((uint64_t)batch * a.G, cols);
        a.prefix_splits = plan_splits(ctx, 2ull * a.prefix_tiles * kv_heads, prefix_len, std::max(128u, 2 * held));
    }
    const uint64_t tasks = plan_own(ctx, a, q_dt, kv_dt, a.G, own_tiles, own_tiles, max_len);
    a.slots = a.prefix_splits + a.splits > 1 ? a.prefix_splits + a.splits : 0;
    // light ones where the own positions weigh as much as the prefix (32 requests of up to
    // 512 behind 4096: 19.7 us against 21.4; of up to 20, 45 behind 10000: 25.7 against 24.7)
    // or are many workgroups (45 of up to 20 at 32/32/128 behind 5000: 25.5 against 29.3)
    a.light = q_dt == JANUS_DT_F16 && hd == 128 && cols >= 64 &&
              (own_tiles * kv_heads >= 2u * (uint32_t)ctx->num_cus || (uint64_t)batch * max_len >= prefix_len);
    return run(ctx, a, q_dt, kv_dt, hd, tasks);
}

}  // namespace janus
