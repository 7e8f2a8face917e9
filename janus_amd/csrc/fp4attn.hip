// fp4attn.hip -- causal attention of packed rows over a KV cache of 4-bit values
// (kvfp4.hip): decode steps, drafted tokens, prompts.
//
// The queries of a KV head that read the same K and V are columns of one matrix
// product: column c of a sequence of n rows is query head c % G of its row c / G (G
// heads per KV head). Positions go by in steps, and the running maximum m, the sum l
// and the output O^T stay in registers:
//   S^T = K Q^T (positions x columns), p = 2^(scale log2(e) s - m + bias),
//   l <- l 2^(m_old - m) + sum p,  O^T <- O^T 2^(m_old - m) + V^T P^T.
// Every 4-bit value times its power-of-two scale is a binary16 number, so K and V
// enter the binary16 matrix unit exactly, converted two values an instruction with the
// scale applied. binary16 rows round P to binary16; binary32 rows have q, divided by a
// power of two per column, and P in two binary16 parts (22 bits), small parts first.
// binary16 rows could have the two parts of P as well, for an error of 2.1e-4, that of their own
// rounding, in place of 2.8e-4: 64 single rows behind up to 8000 positions then take 70 to 72 us
// instead of 66, a prompt of 6000 rows 431 instead of 316. Who needs them has binary32 rows.
//
// Two kernels, by the columns of a sequence and KV head:
//   up to 16, and to 64 where workgroups of one or two KV heads all run at once (decode steps, drafted rows): bound by the read of the cache. A
//     wavefront has one KV head and 32 positions at a time, whose 4-bit rows come into LDS
//     as they are. A decode step of 64 sequences of up to 8000 positions, 32 heads on 8, 128
//     dims: 63 us, 4.6 TB/s, what a large copy reaches; one sequence of 8192 positions 15 us, where
//     the two launches and the start of each count; 16 x 5 binary32 rows behind 2500 positions of
//     32 KV heads 36 us, 2.6 TB/s: while a CU is busy it issues 84% of the time, vector instructions 63%.
//   more (prompts): bound by the matrix unit and what feeds it. Four wavefronts of 32 columns, or
//     two pairs of them for up to 64 or where there are few tiles, share K and V, converted once for all of them. A prompt of 6000 rows: 307 to 335 us, 880 to
//     960 TFLOP/s of what the causal mask leaves, where a large matrix product reaches 1184; 20
//     prompts of 3 to 611 rows 54 us, of which the read of q and the write of the output are
//     22: a workgroup has ten steps at most, and its start and end are not hidden.
//     From 17 columns of more heads on that is faster than tiles of 16 columns that each read K and V (12
//     sequences of 20 columns behind 10574 positions 39 and 45 us, 40 of 30 columns behind 600
//     21 and 39; binary32 rows 46 and 47, 27 and 36).
// Where the tiles are few their positions are split into shares and a third kernel joins
// the parts: a second launch of some 5 us.
// One kernel takes all sequences of a call, by the columns that they have in the mean: 63 single rows behind up to 8000
// positions and a chunk of 512 behind 4000 take 180 us in one call, 66 and 76 in two (with 16 single rows and a chunk of
// 512 without a context 157, 35 and 18).
//
// A scale byte above 140 is a block of NaN. The loops count it as a finite scale and note that
// there was one; the scales are then looked through again and what saw such a block is set: every
// output of a column whose positions include a NaN of K, the block's dims where it is V's. A row
// of q with an infinity or NaN gives NaN, as its formula does.
#include <algorithm>
#include <cmath>

#include "internal.h"

namespace janus {
namespace {

typedef _Float16 fh8 __attribute__((ext_vector_type(8)));
typedef float ff4 __attribute__((ext_vector_type(4)));

struct Fp4Args {
    const void *q;                        // [rows][heads][D]
    const uint8_t *kc, *ks, *vc, *vs;     // [cache rows][kv_heads][D / 2] and [D / 32]
    void *out;                            // [rows][heads][D]
    float *part, *part_ml;                // split: [slot][kv_heads][cols][D], and (m, factor, l, b): weights are multiples of 2^(m factor - b)
    uint32_t *meta;                       // split: [rows * G] (first slot, parts | sees nothing << 23 | column << 24)
    const int32_t *q_start, *row_base, *seq_lens;
    uint32_t rows, nseq, heads, kv_heads, G;
    uint32_t cache_rows, max_seq;
    uint32_t cols;                        // columns of a workgroup
    uint32_t hw, ph;                      // its wavefronts: KV heads x position phases (x columns)
    uint32_t head_groups, shares;         // workgroups of a share of the work; shares
    uint32_t target, least, step;         // split: shares to aim at (0: a tile each), their fewest units of `step` positions
    uint32_t slots;                       // split: places for partial results
    uint32_t mean_parts;                  // host: parts of a tile, in the mean
    float scale2;                         // scale * log2(e)
};

__device__ __forceinline__ float groups_max(float v) {   // over the four lanes of a column
    v = fmaxf(v, swap16(v));
    return fmaxf(v, swap32(v));
}
__device__ __forceinline__ float groups_sum(float v) {
    v += swap16(v);
    return v + swap32(v);
}
__device__ __forceinline__ uint32_t groups_umax(uint32_t v) {
    v = max(v, __float_as_uint(swap16(__uint_as_float(v))));
    return max(v, __float_as_uint(swap32(__uint_as_float(v))));
}

// What a sequence is, whatever the tables hold: rows inside [0, rows), positions inside the cache.
struct SeqRows {
    uint32_t row0, n;    // its rows
    uint32_t avail;      // positions that its last row sees
    int32_t first;       // positions that row 0 sees (may be below 1), each row one more than the last
    uint32_t base;       // cache row of position 0 (0 where avail is)
};
__device__ __forceinline__ SeqRows seq_rows(const Fp4Args &a, uint32_t s) {
    SeqRows q{};
    if (s >= a.nseq) return q;
    const uint32_t each = a.rows / a.nseq;
    int32_t r0 = (int32_t)(s * each), r1 = r0 + (int32_t)each;   // rows are below 2^25
    if (a.q_start) {
        r0 = a.q_start[s];
        r1 = a.q_start[s + 1];
    }
    const int32_t given = a.seq_lens ? a.seq_lens[s] : 0x7fffffff;
    const int64_t base = a.row_base ? (int64_t)a.row_base[s] : (int64_t)((uint64_t)s * a.max_seq);
    r0 = min(max(r0, 0), (int32_t)a.rows);
    r1 = min(max(r1, r0), (int32_t)a.rows);
    q.row0 = (uint32_t)r0;
    q.n = (uint32_t)(r1 - r0);
    const int32_t len = max(a.seq_lens ? given : r1 - r0, -(1 << 26));
    q.first = (int32_t)((uint32_t)len + 1u - q.n);   // n > 0 wherever it is used
    const bool inside = base >= 0 && base < (int64_t)a.cache_rows;
    q.base = inside ? (uint32_t)base : 0u;
    q.avail = inside && len > 0 ? min(min((uint32_t)len, a.max_seq), a.cache_rows - q.base) : 0u;
    return q;
}
// Positions that row r of a sequence sees.
__device__ __forceinline__ uint32_t seen_of(const SeqRows &s, uint32_t r) { return (uint32_t)min(max(s.first + (int32_t)r, 0), (int32_t)min(s.avail, 0x7fffffffu)); }

__device__ __forceinline__ uint32_t lane_value(uint32_t v, uint32_t lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)lane); }

// A lane's number that the compiler takes for a new one each time: what follows from it is
// made again for every share of columns and does not hold registers in between.
__device__ __forceinline__ uint32_t fresh_thread() {
    uint32_t t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// What a workgroup works on: columns of a sequence, and positions [from, to) of theirs.
struct Task {
    SeqRows s;
    uint32_t c0;                        // first column
    uint32_t from, to;
    uint32_t slot, first_slot, parts;   // its place among the parts of these columns; 1 part: the result
    bool more;                          // whether the share goes on behind them
    uint32_t quota, s0, start, before;  // split: units of a share; the sequences looked at, units and tiles before them
};

// The work of share `share` that starts `done` units into it; false if there is none.
// Without a split a share is a tile, that is, cols columns of a sequence. Else
// the positions of all tiles, one behind the other in units of a.step, are cut into
// shares of equal length, wherever tiles begin and end: CUs get an equal part of the
// memory's rate, so all have to be given the same amount. (Parts of 840 positions that began
// anew with each of 64 sequences of up to 8000: 93 us, some CUs with three of them and some with two.)
// A share and a tile that meet have the slot share + tile, both counted from 0, of the
// partial results: a step along the positions raises one of them or both.
template <bool SPLIT> __device__ __forceinline__ bool find_task(const Fp4Args &a, uint32_t share, uint32_t &done, Task &w) {
    const uint32_t lane = threadIdx.x & 63u, shift = 31u - (uint32_t)__builtin_clz(a.cols);   // cols is a power of two
    const uint32_t unit = SPLIT ? 31u - (uint32_t)__builtin_clz(a.step) : 0u;                 // and so is step
    SeqRows q;
    // the host has seen to it that all units together are below 2^31
    auto tiles_of = [&]() { return (q.n * a.G + a.cols - 1) >> shift; };
    auto units_of = [&]() { return SPLIT ? max(1u, (q.avail + a.step - 1) >> unit) : 1u; };
    uint32_t quota = 1, s0 = 0, start = 0, before = 0;   // units and tiles before the sequences from s0 on
    if (!SPLIT || done == 0) {
        q = seq_rows(a, lane);
        if constexpr (SPLIT) {
            uint32_t total = tiles_of() * units_of();
#pragma unroll 4
            for (uint32_t s = 64; s < a.nseq; s += 64) {
                q = seq_rows(a, s + lane);
                total += tiles_of() * units_of();
            }
            total = lane_value(scan_dpp(total), 63);
            w.quota = max((total + a.target - 1) / a.target, a.least);
            if (a.nseq > 64) q = seq_rows(a, lane);
        }
    } else {
        s0 = w.s0;
        start = w.start;
        before = w.before;
        q = seq_rows(a, s0 + lane);
    }
    if constexpr (SPLIT) quota = w.quota;
    if (SPLIT && (done >= quota || (uint64_t)share * quota + done >= 0x80000000u)) return false;
    const uint32_t at = share * quota + done;   // units from the first tile on
    for (;;) {
        const uint32_t tiles = tiles_of(), per = units_of();
        const uint32_t upto = start + scan_dpp(tiles * per), upto_tiles = SPLIT ? scan_dpp(tiles) : 0u;
        const uint64_t here = __ballot(at < upto);
        if (here) {
            const uint32_t l = __builtin_amdgcn_readfirstlane((uint32_t)__builtin_ctzll(here));
            w.s.row0 = lane_value(q.row0, l);
            w.s.n = lane_value(q.n, l);
            w.s.avail = lane_value(q.avail, l);
            w.s.first = (int32_t)lane_value((uint32_t)q.first, l);
            w.s.base = lane_value(q.base, l);
            const uint32_t each = lane_value(per, l), all = lane_value(tiles, l);
            const uint32_t first = lane_value(upto, l) - all * each;   // the sequence's first unit
            const uint32_t in = at - first, tile = SPLIT ? in / each : in, off = SPLIT ? in - tile * each : 0u;
            w.c0 = (all - 1 - tile) << shift;   // the last rows see most: they come first
            if constexpr (!SPLIT) {
                w.from = 0;
                w.to = w.s.avail;
                w.parts = 1;
                w.more = false;
                return true;
            }
            const uint32_t n = min(quota - done, each - off);
            w.from = min(off << unit, w.s.avail);
            w.to = min((off + n) << unit, w.s.avail);
            const uint32_t number = before + lane_value(upto_tiles, l) - all + tile;
            const uint32_t u0 = first + tile * each, s_first = u0 / quota, s_last = (u0 + each - 1) / quota;
            w.parts = s_last - s_first + 1;
            w.slot = share + number;
            w.first_slot = s_first + number;
            done += n;
            w.s0 = s0;
            w.start = start;
            w.before = before;
            w.more = done < quota;
            return w.parts == 1 || w.slot < a.slots;   // more tiles than there can be: sequences that overlap
        }
        start = lane_value(upto, 63);
        if constexpr (SPLIT) before += lane_value(upto_tiles, 63);
        if ((s0 += 64) >= a.nseq) return false;
        q = seq_rows(a, s0 + lane);
    }
}

// Bytes of 32 positions of a KV head, as lane 16 g + at uses them: K of the positions at
// and 16 + at; all scales of a position and head in one word, K's of the two positions,
// V's of the (at % 8)-th of the eight positions {4g .., 16 + 4g ..}.
template <int D> struct Raw {
    uint32_t k[2][D / 32];
    uint32_t ks[2], vs;
};

// A tile of 32 ph positions of hw KV heads, whose rows of hw D / 2 bytes lie one behind the
// other in LDS (2 KB a wavefront of K, then of V, for 128 dims). Whole rows are requested, 1 KB an
// instruction: 270000 positions of 8 heads come at 6.4 TB/s like this and at 4.9 where
// every wavefront loads its own head's 64 bytes of a row. The 16-byte segments of a row
// are permuted by the heads' number of segments (U), so that 16 positions of a head (K), or four
// positions four apart (V), lie in different banks.
template <int D, int NW> struct Tile {
    static constexpr uint32_t U = D / 32, kBytes = 16u * NW * D;   // segments of a head; bytes of K
    static constexpr int N = kBytes / (1024 * NW);                  // requests of a wavefront for K
    static constexpr uint32_t kLds = 4 * kBytes;                    // two tiles
    const uint8_t *kc, *ks, *vc, *vs;   // of the workgroup's first head at position 0
    uint32_t row, srow;                 // bytes from a position to the next
    uint32_t segs, heads, fold;         // segments of a row of the tile; hw - 1; log2 of the positions in 256 bytes
    uint32_t ko[N], vo[N];              // of the lane, from the tile's first position

    __device__ __forceinline__ uint32_t k_turn(uint32_t pos) const { return (pos >> fold & heads) * U; }
    __device__ __forceinline__ uint32_t v_turn(uint32_t pos) const { return (pos >> 2 & heads) * U; }
    // The lane's offsets, positions from `last` on repeated.
    __device__ __forceinline__ void offsets(uint32_t lane, uint32_t wave, uint32_t last) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t slot = (wave * N + i) * 64u + lane, pos = slot / segs, seg = slot & (segs - 1), n = min(pos, last);
            ko[i] = n * row + (seg ^ k_turn(pos)) * 16u;
            vo[i] = n * row + (seg ^ v_turn(pos)) * 16u;
        }
    }
    __device__ __forceinline__ void request(uint32_t p, uint32_t wave, uint32_t lds) const {
        const uint8_t *kp = kc + (size_t)p * row, *vp = vc + (size_t)p * row;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            lds_request<true>(kp, ko[i], lds + (wave * N + i) * 1024u);
            lds_request<true>(vp, vo[i], lds + kBytes + (wave * N + i) * 1024u);
        }
    }
};

// High bit of every byte above 140.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x73737373u) & w & 0x80808080u; }
__device__ __forceinline__ uint32_t without_nans(uint32_t w) {
    const uint32_t m = (nan_bytes(w) >> 7) * 255u;
    return (w & ~m) | (m & 0x7f7f7f7fu);
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(min(byte, 140u) << 23); }

template <int BYTE> __device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, BYTE));
}

__device__ __forceinline__ fh8 h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(fh8, make_uint4(a, b, c, d));
}
__device__ __forceinline__ uint32_t half_pair(float a, float b) {
    jh2 h = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, h);
}
__device__ __forceinline__ ff4 mfma(fh8 a, fh8 b, ff4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// The factor from scores to exponents: not 0, since it also multiplies -infinity, nor infinite (a scale or a row of q
// near the end of binary32), since it also multiplies differences of 0. The limits change no weight: scores, as the
// products have them, are whole multiples of 2^-48 and below 2^39.
__device__ __forceinline__ float finite_factor(float cs) { return fminf(fmaxf(cs, 1e-37f), 3e38f); }

// Sixteen columns of a wavefront. Lane 16 g + a:
//   K: its bytes of a position lie in one block of 32 dims, and the order of dims in the sum is
//     free, so D / 8 consecutive bytes are its operand of the D / 32 products;
//   S -> P: the result layout of two score tiles (16 positions each) is the operand layout of 32
//     positions, in the order {4g .. 4g + 3, 16 + 4g .. 16 + 4g + 3}; V takes its positions in
//     the same order;
//   V: it reads dims [a D / 16, (a + 1) D / 16) of its eight positions; product i takes dim i of
//     every lane's, after pairs of positions are put together (v_perm).
// Its outputs are D / 4 consecutive dims of column a.
template <typename T, int D> struct Columns {
    static constexpr int P = sizeof(T) == 4 ? 2 : 1;   // binary16 parts of q and of P
    // The maximum may grow by kSlack powers of two before anything is rescaled; p, up to
    // 2^(kBias + kSlack), stays finite in binary16, and small ones normal (in two parts the
    // second is off by 2^-25 of 2^kBias).
    static constexpr float kBias = P == 2 ? 13.0f : 7.0f, kSlack = P == 2 ? 2.0f : 8.0f;
    fh8 q[P][D / 32];
    float cs;                       // factor from s to the exponent
    float m, l;
    ff4 o[D / 16];
    uint32_t vis;                   // positions that the lane's column sees
    bool bad;                       // the column has an infinity or NaN in q

    __device__ __forceinline__ void load(const Fp4Args &a, const Task &w, uint32_t lane, uint32_t c0, uint32_t kvh) {
        const uint32_t g = lane >> 4;
        bad = false;
        const uint32_t c = c0 + (lane & 15u), row = c / a.G;   // below 2^25
        const bool there = row < w.s.n;
        vis = 0;
        float x[D / 4];
        uint32_t top = 0;
        if (there) {
            vis = seen_of(w.s, row);
            const T *src = (const T *)a.q + ((size_t)(w.s.row0 + row) * a.heads + (size_t)kvh * a.G + (c - row * a.G)) * D + g * (D / 4);
            typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
            for (int i = 0; i < D / 4; i += 16 / (int)sizeof(T)) {
                const vec v = *(const vec *)(src + i);
#pragma unroll
                for (int j = 0; j < 16 / (int)sizeof(T); ++j) x[i + j] = (float)v[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < D / 4; ++i) x[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < D / 4; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        top = groups_umax(top);
        if (top >= 0x7f800000u) {
            bad = true;
            top = 0;
#pragma unroll
            for (int i = 0; i < D / 4; ++i) x[i] = 0.0f;
        }
        if constexpr (P == 1) {
            cs = a.scale2;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
                q[0][i] = h8(half_pair(x[8 * i], x[8 * i + 1]), half_pair(x[8 * i + 2], x[8 * i + 3]),
                                half_pair(x[8 * i + 4], x[8 * i + 5]), half_pair(x[8 * i + 6], x[8 * i + 7]));
        } else {
            // the column's largest into [2^14, 2^15): the second part of what is 2^-17 of it is subnormal, off by 2^-39 of it
            const int e = max((int)(top >> 23), 1) - 127 - 14;
            cs = ldexpf(a.scale2, e);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                fh8 hi, lo;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float y = ldexpf(x[8 * i + j], -e);
                    hi[j] = (_Float16)y;
                    lo[j] = (_Float16)(y - (float)hi[j]);
                }
                q[0][i] = hi;
                q[1][i] = lo;
            }
        }
        cs = finite_factor(cs);
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i] = ff4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // 32 positions from p on. masked: some column of the wavefront does not see all of
    // them. v(j): the lane's bytes of V at its position j. Returns whether a block among
    // them is NaN; its scale counts as 1 then.
    template <typename V> __device__ __forceinline__ bool step(Raw<D> &r, uint32_t lane, uint32_t p, bool masked, V v) {
        const uint32_t g = lane >> 4;
        const bool odd = __any((nan_bytes(r.ks[0]) | nan_bytes(r.ks[1]) | nan_bytes(r.vs)) != 0);
        if (odd) {
            r.ks[0] = without_nans(r.ks[0]);
            r.ks[1] = without_nans(r.ks[1]);
            r.vs = without_nans(r.vs);
        }
        const uint32_t kshift = g * (D / 4) / 32 * 8;   // the lane's block of K, and of V
        const uint32_t vblock = (lane & 15u) * (D / 16) / 32, vmask = 0xffu << (8u * vblock), vturn = (8u * vblock - 23u) & 31u;
        ff4 s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float sc = __uint_as_float((r.ks[h] >> kshift & 0xffu) << 23);
            ff4 small = {};
            s[h] = ff4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const uint32_t w = r.k[h][i];
                const fh8 k = h8(fp4_pair<0>(w, sc), fp4_pair<1>(w, sc), fp4_pair<2>(w, sc), fp4_pair<3>(w, sc));
                if constexpr (P == 2) small = mfma(k, q[1][i], small);
                s[h] = mfma(k, q[0][i], s[h]);
            }
            if constexpr (P == 2) s[h] += small;
        }
        if (masked) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[h][j] = p + 16u * h + 4u * g + j < vis ? s[h][j] : -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int j = 1; j < 8; ++j) mx = fmaxf(mx, s[j >> 2][j & 3]);
        mx = groups_max(mx);
        if (__any((mx - m) * cs > kSlack)) {
            const float now = fmaxf(m, mx);
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - now) * cs);
            l *= f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[i] *= f;
            m = now;
        }
        const float m0 = m == -INFINITY ? 0.0f : m;
        fh8 pp[P];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = __builtin_amdgcn_exp2f(fmaf(s[j >> 2][j & 3] - m0, cs, kBias));   // large scores keep their last bits
            pp[0][j] = (_Float16)x;
            if constexpr (P == 2) {
                l += x;
                pp[1][j] = (_Float16)(x - (float)pp[0][j]);
            }
        }
        if constexpr (P == 1) {   // of P as rounded: both sums see the same weights
            const jh2 one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
            for (int j = 0; j < 8; j += 2) l = __builtin_amdgcn_fdot2(jh2{pp[0][j], pp[0][j + 1]}, one, l, false);
        }
        // the byte of position j, which lane j of the 16 holds, at the exponent's place
        float sc[8];
        auto spread = [&](auto j) {
            const uint32_t w = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)r.vs, 0x150 + decltype(j)::value, 0xf, 0xf, false) & vmask;   // row_newbcast
            sc[decltype(j)::value] = __uint_as_float(__builtin_amdgcn_alignbit(w, w, vturn));
        };
        spread(std::integral_constant<int, 0>{});
        spread(std::integral_constant<int, 1>{});
        spread(std::integral_constant<int, 2>{});
        spread(std::integral_constant<int, 3>{});
        spread(std::integral_constant<int, 4>{});
        spread(std::integral_constant<int, 5>{});
        spread(std::integral_constant<int, 6>{});
        spread(std::integral_constant<int, 7>{});
        uint32_t raw[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) raw[j] = v(j);
        auto two = [&](auto byte) {
            constexpr int B = decltype(byte)::value;
            uint32_t h[8], lo[4], hi[4];
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = fp4_pair<B>(raw[j], sc[j]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                lo[j] = __builtin_amdgcn_perm(h[2 * j + 1], h[2 * j], 0x05040100u);
                hi[j] = __builtin_amdgcn_perm(h[2 * j + 1], h[2 * j], 0x07060302u);
            }
            const fh8 v0 = h8(lo[0], lo[1], lo[2], lo[3]), v1 = h8(hi[0], hi[1], hi[2], hi[3]);
#pragma unroll
            for (int w = 0; w < P; ++w) {
                o[2 * B] = mfma(v0, pp[w], o[2 * B]);
                o[2 * B + 1] = mfma(v1, pp[w], o[2 * B + 1]);
            }
        };
        two(std::integral_constant<int, 0>{});
        two(std::integral_constant<int, 1>{});
        if constexpr (D == 128) {
            two(std::integral_constant<int, 2>{});
            two(std::integral_constant<int, 3>{});
        }
        return odd;
    }
};

// First positions with a NaN block of K (x), and of V in the lane's output dims (y),
// among 32 positions from each of p, p + step, ... below end.
template <int D>
__device__ __forceinline__ uint2 first_nans(const uint8_t *ks, const uint8_t *vs, uint32_t srow, uint32_t p, uint32_t end,
                                            uint32_t step) {
    const uint32_t lane = threadIdx.x & 63u, mine = (lane >> 4) * (D / 4) / 32;
    uint2 at = make_uint2(0xffffffffu, 0xffffffffu);
    for (; p < end; p += step) {
        const uint32_t i = p + lane;
        bool kn = false;
        for (uint32_t b = 0; b < D / 32; ++b) {
            bool vn = false;
            if (lane < 32u && i < end) {
                kn |= ks[(size_t)i * srow + b] > 140;
                vn = vs[(size_t)i * srow + b] > 140;
            }
            const uint64_t some = __ballot(vn);
            if (some && b == mine) at.y = min(at.y, p + (uint32_t)__builtin_ctzll(some));
        }
        const uint64_t some = __ballot(kn);
        if (some) at.x = min(at.x, p + (uint32_t)__builtin_ctzll(some));
    }
    return at;
}

// A tile of up to 16 columns of a sequence and positions [from, to): the NW wavefronts of a
// workgroup take hw KV heads and ph phases of 32 positions each; PER of them share a SIMD.
template <typename T, int D, int NW, int PER, bool SPLIT>
__global__ __launch_bounds__(NW * 64, PER) void fp4_attn_kernel(Fp4Args args) {
    constexpr uint32_t DL = D / 4;   // output dims of a lane
    extern __shared__ __align__(16) uint8_t smem[];   // two tiles, then the phases' results
    float *const lds = (float *)smem;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)smem;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // the head groups of a share one behind the other on one XCD (workgroup b runs on XCD b % 8): they share lines of the scales
    const uint32_t j = blockIdx.x >> 3;
    const uint32_t share = j / args.head_groups * 8u + (blockIdx.x & 7u);
    if (share >= args.shares) return;
    Task w;
    w.more = true;
    for (uint32_t done = 0; w.more && find_task<SPLIT>(late_args<Fp4Args>(), share, done, w);) {
        const Fp4Args &a = late_args<Fp4Args>();
        const uint32_t lane = fresh_thread() & 63u, g = lane >> 4, at = lane & 15u;
        const uint32_t hwave = wave & (a.hw - 1), phase = wave / a.hw, head0 = (blockIdx.x >> 3) % a.head_groups * a.hw, kvh = head0 + hwave;
        const uint32_t c0 = w.c0, columns = w.s.n * a.G;   // below 2^25

        // positions that columns of the tile see: the last ones the most
        const uint32_t most = seen_of(w.s, (min(c0 + 16u, columns) - 1) / a.G), fewest = seen_of(w.s, c0 / a.G);
        const uint32_t end = __builtin_amdgcn_readfirstlane(min(most, w.to)), from = __builtin_amdgcn_readfirstlane(w.from), step = 32u * a.ph;
        const size_t base = w.s.base;
        const uint32_t rows = a.cache_rows - w.s.base;   // of the cache from position 0 on
        Tile<D, NW> tile;
        tile.row = a.kv_heads * (D / 2);
        tile.srow = a.kv_heads * (D / 32);
        tile.kc = a.kc + base * tile.row + head0 * (D / 2);
        tile.vc = a.vc + base * tile.row + head0 * (D / 2);
        tile.ks = a.ks + base * tile.srow + kvh * (D / 32);   // the wavefront's own
        tile.vs = a.vs + base * tile.srow + kvh * (D / 32);
        tile.segs = a.hw * Tile<D, NW>::U;
        tile.heads = a.hw - 1;
        tile.fold = tile.segs >= 16u ? 0u : 4u - (31u - (uint32_t)__builtin_clz(tile.segs));
        tile.offsets(lane, wave, step - 1);
        // the scales of the wavefront's 32 positions of a tile
        typedef std::conditional_t<D == 128, uint32_t, uint16_t> word;
        uint32_t ks0 = 0, ks1 = 0, vs0 = 0;
        const uint32_t kpos = at, vpos = (at & 4u) * 4u + 4u * g + (at & 3u);
        const uint32_t kso = kpos * tile.srow, vso = vpos * tile.srow;
        auto fetch = [&](uint32_t p, uint32_t b) {
            const uint32_t q = p + 32u * phase;
            if (p + step > rows) {   // the cache ends inside the tile: its last row again
                tile.offsets(lane, wave, rows - 1 - p);
                tile.request(p, wave, lds0 + b * (2 * Tile<D, NW>::kBytes));
                ks0 = *(const word *)(tile.ks + (size_t)min(q + kpos, rows - 1) * tile.srow);
                ks1 = *(const word *)(tile.ks + (size_t)min(q + kpos + 16u, rows - 1) * tile.srow);
                vs0 = *(const word *)(tile.vs + (size_t)min(q + vpos, rows - 1) * tile.srow);
                return;
            }
            // rows behind the sequence's end are other sequences' or none's, and no column sees them
            tile.request(p, wave, lds0 + b * (2 * Tile<D, NW>::kBytes));
            ks0 = *(const word *)(tile.ks + (size_t)q * tile.srow + kso);
            ks1 = *(const word *)(tile.ks + (size_t)(q + 16u) * tile.srow + kso);
            vs0 = *(const word *)(tile.vs + (size_t)q * tile.srow + vso);
        };
        if (from < end) fetch(from, 0);
        Columns<T, D> col;
        col.load(a, w, lane, c0, kvh);
        if (from < end) {
            bool odd = false;
            // offsets of the lane's operands in a tile: K of position at of 16, V of 4 g of 16 (r rows on under the same turn)
            const uint32_t pos0 = 32u * phase, seg0 = hwave * Tile<D, NW>::U, line = tile.segs * 16u;
            uint32_t kat[2], vat[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t kn = pos0 + 16u * h + at, vn = pos0 + 16u * h + 4u * g;
                kat[h] = kn * line + ((seg0 + g * (D / 8) / 16) ^ tile.k_turn(kn)) * 16u + (D == 64 ? (g & 1u) * 8u : 0u);
                vat[h] = vn * line + ((seg0 + at * (D / 32) / 16) ^ tile.v_turn(vn)) * 16u + at * (D / 32) % 16u;
            }
            uint32_t b = 0;
            for (uint32_t p = from; p < end; p += step, b ^= 1u) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();   // this tile is there, the other one has been read
                Raw<D> r;
                // the scales are in registers before the next ones are asked for: a wait for them later would be one for the next tile too
                r.ks[0] = ks0;
                r.ks[1] = ks1;
                r.vs = vs0;
                asm volatile("" : "+v"(r.ks[0]), "+v"(r.ks[1]), "+v"(r.vs));
                if (p + step < end) fetch(p + step, b ^ 1u);
                const uint32_t mine = p + 32u * phase;
                if (mine >= end) continue;
                const uint8_t *kt = smem + b * (2 * Tile<D, NW>::kBytes), *vt = kt + Tile<D, NW>::kBytes;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    typedef uint32_t vec __attribute__((ext_vector_type(D / 32)));
                    const vec k = *(const vec *)(kt + kat[h]);
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) r.k[h][i] = k[i];
                }
                odd |= col.step(r, lane, mine, mine + 32u > fewest || mine + 32u > end,
                                [&](int j) -> uint32_t { return *(const word *)(vt + vat[j >> 2] + (j & 3) * line); });
            }
            if (odd) {
                const uint2 at = first_nans<D>(tile.ks, tile.vs, tile.srow, from + 32u * phase, end, step);
                const float nan = __uint_as_float(0x7fc00000u);
                if (at.x < col.vis) col.l = nan;
                if (at.y < col.vis)
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) col.o[i] = ff4{nan, nan, nan, nan};
            }
        }

        if (SPLIT || a.ph > 1) __syncthreads();   // the tiles have been read
        // the phases of a head and column tile join in its first one
        col.l = groups_sum(col.l);
        if (a.ph > 1) {
            constexpr uint32_t kArea = (D / 4 + 2) * 64u;   // floats of a wavefront
            float *mine = lds + ((phase - 1) * a.hw + hwave) * kArea;
            if (phase > 0) {
                float *at = mine + lane;
                at[0] = col.m;
                at[64] = col.l;
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) at[(2 + 4 * i + r) * 64] = col.o[i][r];
            }
            __syncthreads();
            for (uint32_t h = 1; phase == 0 && h < a.ph; ++h) {
                const float *at = lds + ((h - 1) * a.hw + hwave) * kArea + lane;
                const float m2 = at[0], now = fmaxf(col.m, m2);
                const float f1 = col.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((col.m - now) * col.cs);
                const float f2 = m2 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m2 - now) * col.cs);
                // what has seen nothing is 0, or NaN where a block was marked
                col.l = col.l * f1 + at[64] * f2;
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) col.o[i][r] = col.o[i][r] * f1 + at[(2 + 4 * i + r) * 64] * f2;
                col.m = now;
            }
            if constexpr (SPLIT) __syncthreads();   // the areas are written again for the next columns
            if (phase > 0) {
                if constexpr (SPLIT) continue;
                else return;
            }
        }
        const Fp4Args &z = late_args<Fp4Args>();
        const uint32_t c = c0 + (lane & 15u);
        if (c < columns) {   // no lane leaves the loop: the search for the next columns needs all
            const uint32_t r = c / z.G, gh = c % z.G;
            if (col.bad && col.vis) col.l = __uint_as_float(0x7fc00000u);
            if (SPLIT && w.parts > 1) {
                const size_t at = ((size_t)w.slot * z.kv_heads + kvh) * z.cols + (c - w.c0);
                float *to = z.part + at * D + g * DL;
#pragma unroll
                for (int rr = 0; rr < 4; ++rr)
#pragma unroll
                    for (int i = 0; i < D / 16; i += 4)
                        *(ff4 *)(to + rr * (D / 16) + i) = ff4{col.o[i][rr], col.o[i + 1][rr], col.o[i + 2][rr], col.o[i + 3][rr]};
                if (g == 0) *(ff4 *)(z.part_ml + 4 * at) = ff4{col.m, col.cs, col.l, 0.0f};   // kBias, in all parts alike, counts for nothing
            } else {
                const float inv = col.vis ? 1.0f / col.l : 0.0f;
                T *to = (T *)z.out + ((size_t)(w.s.row0 + r) * z.heads + (size_t)kvh * z.G + gh) * D + g * DL;
#pragma unroll
                for (int rr = 0; rr < 4; ++rr) {
                    typedef T vec __attribute__((ext_vector_type(D / 16 * sizeof(T) > 16 ? 4 : D / 16)));
                    constexpr int N = sizeof(vec) / sizeof(T);
#pragma unroll
                    for (int i = 0; i < D / 16; i += N) {
                        vec v;
#pragma unroll
                        for (int u = 0; u < N; ++u) v[u] = col.vis ? (T)(col.o[i + u][rr] * inv) : (T)0.0f;
                        *(vec *)(to + rr * (D / 16) + i) = v;
                    }
                }
            }
            if (SPLIT && w.slot == w.first_slot && kvh == 0 && g == 0) {
                uint32_t *to = z.meta + 2 * ((size_t)w.s.row0 * z.G + c);
                to[0] = w.first_slot;
                to[1] = w.parts | (col.vis ? 0u : 1u << 23) | (c - w.c0) << 24;
            }
        }
    }
}

// Joins the parts of a row and head: W wavefronts take them in turn, eight at a time,
// and are joined themselves. Workgroups of 4 units for W = 1, else of one. The exponents m factor - b
// are exact in binary64: in 32 bits their rounding would be that of the parts' weights.
template <typename T, int D, int W> __global__ __launch_bounds__(W == 1 ? 256 : W * 64) void fp4_join_kernel(Fp4Args a) {
    __shared__ double sm[W];
    __shared__ float sl[W], so[W][D];
    const uint32_t lane = threadIdx.x & 63u, wave = W == 1 ? 0u : threadIdx.x >> 6;
    const uint32_t unit = __builtin_amdgcn_readfirstlane(W == 1 ? blockIdx.x * 4u + (threadIdx.x >> 6) : blockIdx.x);
    const uint32_t row = unit / a.heads, head = unit - row * a.heads;
    if (row >= a.rows) return;
    const uint32_t kvh = head / a.G, gh = head - kvh * a.G;
    const uint2 meta = *(const uint2 *)(a.meta + 2 * ((size_t)row * a.G + gh));
    if (a.q_start) {   // a row of no sequence: what meta holds is not its own
        bool mine = false;
        for (uint32_t s = lane; s < a.nseq; s += 64) mine |= a.q_start[s] <= (int32_t)row && (int32_t)row < a.q_start[s + 1];
        if (!__any(mine)) return;
    }
    const uint32_t first = meta.x, parts = meta.y & 0x7fffffu, c = meta.y >> 24;
    const bool sees = !(meta.y >> 23 & 1u);
    if (parts < 2 || (uint64_t)first + parts > a.slots || c >= a.cols) return;
    constexpr int E = D / 64;
    typedef float vec __attribute__((ext_vector_type(E)));
    const size_t stride = (size_t)a.kv_heads * a.cols;
    const size_t at0 = ((size_t)first * a.kv_heads + kvh) * a.cols + c;
    double m = -INFINITY;
    float l = 0.0f;
    vec o = {};
    for (uint32_t i0 = wave * 8; i0 < parts; i0 += W * 8) {
        ff4 ml[8];
        double e[8];
        vec po[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const size_t at = at0 + (size_t)min(i0 + i, parts - 1) * stride;
            ml[i] = *(const ff4 *)(a.part_ml + 4 * at);
            po[i] = *(const vec *)(a.part + at * D + lane * E);
        }
        double now = m;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            e[i] = i0 + i < parts ? (double)ml[i][0] * (double)ml[i][1] - (double)ml[i][3] : -INFINITY;
            now = fmax(now, e[i]);
        }
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((float)(m - now));
        l *= f;
        o *= f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float fi = e[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((float)(e[i] - now));
            // a part that has seen nothing holds zeros, or NaN where a block was marked
            if (i0 + i < parts) {
                l += ml[i][2] * fi;
                o += po[i] * fi;
            }
        }
        m = now;
    }
    T *out = (T *)a.out + ((size_t)row * a.heads + head) * D;
    if constexpr (W == 1) {
        const float inv = 1.0f / l;
#pragma unroll
        for (int e = 0; e < E; ++e) out[lane * E + e] = sees ? (T)(o[e] * inv) : (T)0.0f;
    } else {
        if (lane == 0) {
            sm[wave] = m;
            sl[wave] = l;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) so[wave][lane * E + e] = o[e];
        __syncthreads();
        if (threadIdx.x >= D) return;
        double now = sm[0];
#pragma unroll
        for (int i = 1; i < W; ++i) now = fmax(now, sm[i]);
        float total = 0.0f, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float f = sm[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((float)(sm[i] - now));
            total += sl[i] * f;
            sum += so[i][threadIdx.x] * f;
        }
        out[threadIdx.x] = sees ? (T)(sum / total) : (T)0.0f;
    }
}

// ---- many columns -----------------------------------------------------------------
//
// Wavefronts of 32 columns share K and V: tiles of TP positions are loaded in 4 bits
// into registers two tiles ahead, converted one tile ahead and written to LDS as
// the operands of v_mfma_f32_32x32x16_f16 that they will be, 16 bytes a lane, so that every
// wavefront reads them in a straight line.
//   K: operand (position n, dims 16 s + 8 h ..) at slot ((n / 32) D / 16 + s) 64 + 32 h + n % 32
//   S^T: position 8 (v / 4) + 4 h + v % 4 of column lane % 32 in s[v], h = lane / 32, which is
//     the operand order of 16 positions for P;
//   V: operand (dim i, positions 4 h .. and 8 + 4 h .. of 16) at slot (.. D / 32 + i / 32) 64 + 32 h + i % 32;
//     a lane converts four positions of 8 dims and writes 8 bytes of each; the slots of 8
//     dims are permuted by the dims' number so that lanes meet different banks.

// First positions of a NaN block of K, and of V by block, among [p, end).
template <int D> struct Nans {
    uint32_t k, v[D / 32];
};
template <int D> __device__ __forceinline__ Nans<D> all_nans(const uint8_t *ks, const uint8_t *vs, uint32_t srow, uint32_t p, uint32_t end) {
    const uint32_t lane = threadIdx.x & 63u;
    Nans<D> at;
    at.k = 0xffffffffu;
#pragma unroll
    for (int b = 0; b < D / 32; ++b) at.v[b] = 0xffffffffu;
    for (; p < end; p += 64) {
        const uint32_t i = p + lane;
        bool kn = false;
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
            bool vn = false;
            if (i < end) {
                kn |= ks[(size_t)i * srow + b] > 140;
                vn = vs[(size_t)i * srow + b] > 140;
            }
            const uint64_t some = __ballot(vn);
            if (some) at.v[b] = min(at.v[b], p + (uint32_t)__builtin_ctzll(some));
        }
        const uint64_t some = __ballot(kn);
        if (some) at.k = min(at.k, p + (uint32_t)__builtin_ctzll(some));
    }
    return at;
}

// A wavefront's 32 rows of q or of the output pass through LDS, so that memory sees whole
// lines: a lane has (needs) 16 or 8 bytes of a row at a time, and 32 rows' next ones.
// Rows of `Rows::kBytes` bytes, their 16-byte pieces permuted by the row's number.
template <typename T, int D, int TP> struct Rows {
    static constexpr uint32_t kBytes = TP * D / 32, kPieces = kBytes / 16, kDims = kBytes / sizeof(T);
    static constexpr int kPasses = D * sizeof(T) / kBytes, kTurns = kPieces / 2;   // 64 pieces a turn
    static_assert(kBytes >= 128 && kPasses * kDims == D, "whole lines");
    static __device__ __forceinline__ uint32_t place(uint32_t row, uint32_t piece) {
        return row * kBytes + (piece ^ ((kPieces == 16 ? row : row >> 1) & (kPieces - 1))) * 16u;
    }
};

// PH 1: four wavefronts of 32 columns. PH 2: two, with two wavefronts each, which take every
// other 32 positions and are joined at the end: for up to 64 columns of a sequence, where two of
// four wavefronts or more would have none, and for few tiles (12 binary32 sequences of 40 columns behind 10574 positions 53 us,
// 66 with PH 1; 40 binary16 ones behind 600 23 and 27; one of 20 columns 18.5 and 18).
template <typename T, int D, int TP, int PH, bool SPLIT>
__global__ __launch_bounds__(256, 2) void fp4_wide_kernel(Fp4Args args) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1, NB = TP / 32 / PH, QN = D / 16, ND = D / 32;   // NB: of a wavefront
    constexpr uint32_t kCols = 128 / PH;
    constexpr float kBias = P == 2 ? 13.0f : 7.0f, kSlack = P == 2 ? 2.0f : 8.0f;
    constexpr uint32_t kTile = TP * D * 2u;   // bytes of a tile of K, and of V
    constexpr uint32_t kUnits = TP * D / 32;  // 16-byte pieces of K, and quads of positions x 8 dims of V
    static_assert(kUnits == 256 || kUnits == 128, "a lane has one unit of each, or of one of them");
    extern __shared__ __align__(16) uint8_t smem[];         // K, V, K, V
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // KV heads change fastest, so with eight of them an XCD's L2 holds the lines of one or two
    const uint32_t share = blockIdx.x / args.kv_heads, kvh = blockIdx.x % args.kv_heads;
    Task w;
    w.more = true;
    for (uint32_t done = 0; w.more && find_task<SPLIT>(late_args<Fp4Args>(), share, done, w);) {
        const Fp4Args &a = late_args<Fp4Args>();
        const uint32_t tid = fresh_thread(), lane = tid & 63u, col = lane & 31u, h = lane >> 5;
        const uint32_t columns = w.s.n * a.G;
        auto seen = [&](uint32_t c) { return seen_of(w.s, c / a.G); };
        const uint32_t group_hi = seen(min(w.c0 + kCols - 1, columns - 1));   // the last column sees most
        const uint32_t p0 = __builtin_amdgcn_readfirstlane(min(w.from, group_hi)), p1 = __builtin_amdgcn_readfirstlane(min(w.to, group_hi));
        const uint32_t phase = PH == 1 ? 0u : wave >> 1;
        const uint32_t c0 = w.c0 + 32u * (PH == 1 ? wave : wave & 1u);
        const bool idle = c0 >= columns;
        const uint32_t wave_lo = idle ? 0u : __builtin_amdgcn_readfirstlane(seen(c0));
        const uint32_t wave_hi = idle ? 0u : __builtin_amdgcn_readfirstlane(min(seen(min(c0 + 31u, columns - 1)), p1));
        const uint32_t c = min(c0 + col, columns - 1), vis = seen(c);
        const uint32_t qat = (w.s.row0 + c / a.G) * a.heads + kvh * a.G + c % a.G;   // rows * heads is below 2^25

        const uint32_t row = a.kv_heads * (D / 2), srow = a.kv_heads * (D / 32);
        const size_t base = w.s.base;
        const uint8_t *kc = a.kc + base * row + kvh * (D / 2), *ks = a.ks + base * srow + kvh * (D / 32);
        const uint8_t *vc = a.vc + base * row + kvh * (D / 2), *vs = a.vs + base * srow + kvh * (D / 32);

        // what a lane loads of a tile: block kb of position kn of K, and dims 8 vd .. of positions 4 vq .. of V
        const uint32_t ku = tid, vu = kUnits == 256 ? tid : tid ^ 128u;
        const bool has_k = kUnits == 256 || ku < kUnits, has_v = kUnits == 256 || vu < kUnits;
        const uint32_t kn = (ku & 15u) + ku / (D / 2) * 16u, kb = ku / 16u % (D / 32), vd = vu % (D / 8), vq = vu / (D / 8);
        ju4 kr;
        uint32_t ksr = 0, vr[4], vsr[4] = {};
        uint32_t ko, kso, vo[4], vso[4];   // offsets of a lane's bytes from the tile's first position
        auto offsets = [&](uint32_t last) {   // rows beyond the part repeat its last one
            const uint32_t n = min(kn, last);
            ko = n * row + kb * 16u;
            kso = n * srow + kb;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t n = min(4u * vq + i, last);
                vo[i] = n * row + vd * 4u;
                vso[i] = n * srow + vd / 4u;
            }
        };
        offsets(min((uint32_t)TP, p1 - p0) - 1);
        auto load = [&](uint32_t p) {
            if (p + TP > p1) offsets(p1 - 1 - p);
            const uint8_t *kp = kc + (size_t)p * row, *ksp = ks + (size_t)p * srow, *vp = vc + (size_t)p * row, *vsp = vs + (size_t)p * srow;
            if (has_k) {
                kr = *(const ju4 *)(kp + ko);
                ksr = ksp[kso];
            }
            if (has_v)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    vr[i] = *(const uint32_t *)(vp + vo[i]);
                    vsr[i] = vsp[vso[i]];
                }
        };
        uint32_t worst = 0;
        auto store = [&](uint32_t b) {
            uint8_t *kt = smem + b * 2 * kTile, *vt = kt + kTile;
            if (has_k) {
                const float sc = scale_of(ksr);
                worst = max(worst, ksr);
                uint8_t *to = kt + ((kn / 32 * QN + 2 * kb) * 64u + kn % 32) * 16u;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *(ju4 *)(to + ((i >> 1) * 64u + (i & 1) * 32u) * 16u) =
                        ju4{fp4_pair<0>(kr[i], sc), fp4_pair<1>(kr[i], sc), fp4_pair<2>(kr[i], sc), fp4_pair<3>(kr[i], sc)};
            }
            if (has_v) {
                float sc[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[i] = scale_of(vsr[i]);
                    worst = max(worst, vsr[i]);
                }
                // block vd / 4, slots 8 (vd % 4) .. of its 32; quad vq % 4: half vq % 2, first or second 8 bytes
                uint8_t *to = vt + ((vq / 4 * ND + vd / 4) * 64u + (vq & 1u) * 32u + (vd & 3u) * 8u) * 16u + (vq >> 1 & 1u) * 8u;
                const uint32_t turn = (vd & 7u) * 16u;
                auto two = [&](auto byte) {
                    constexpr int B = decltype(byte)::value;
                    uint32_t x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = fp4_pair<B>(vr[i], sc[i]);
                    *(uint2 *)(to + ((2 * B * 16u) ^ turn)) = make_uint2(__builtin_amdgcn_perm(x[1], x[0], 0x05040100u), __builtin_amdgcn_perm(x[3], x[2], 0x05040100u));
                    *(uint2 *)(to + (((2 * B + 1) * 16u) ^ turn)) = make_uint2(__builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u));
                };
                two(std::integral_constant<int, 0>{});
                two(std::integral_constant<int, 1>{});
                two(std::integral_constant<int, 2>{});
                two(std::integral_constant<int, 3>{});
            }
        };
        const uint32_t last_tile = p0 + (p1 > p0 ? (p1 - p0 - 1) / TP * TP : 0u);
        if (p0 < p1) load(p0);

        // q of the lane's column
        fh8 q[P][QN];
        float cs = a.scale2;
        bool bad = false;
        {
            float x[QN][8];
            uint32_t top = 0;
            typedef Rows<T, D, TP> R;
            uint8_t *const stage = smem + 2 * kTile + wave * (32u * R::kBytes);   // of the second tile, which nobody writes before the loop's first barrier
            const uint32_t piece = lane % R::kPieces, r0 = lane / R::kPieces;
            ju4 raw[R::kPasses][R::kTurns];
#pragma unroll
            for (int i = 0; i < R::kTurns; ++i) {
                const T *src = (const T *)a.q + (size_t)__shfl(qat, (int)(r0 + i * (64u / R::kPieces))) * D + piece * (16 / sizeof(T));
#pragma unroll
                for (int k = 0; k < R::kPasses; ++k) raw[k][i] = *(const ju4 *)(src + k * R::kDims);
            }
#pragma unroll
            for (int k = 0; k < R::kPasses; ++k) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (int i = 0; i < R::kTurns; ++i) *(ju4 *)(stage + R::place(r0 + i * (64u / R::kPieces), piece)) = raw[k][i];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (int s = 0; s < QN / R::kPasses; ++s) {
                    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
                    for (int i = 0; i < 8; i += 16 / (int)sizeof(T)) {
                        const vec v = *(const vec *)(stage + R::place(col, (16u * s + 8u * h + i) * sizeof(T) / 16u));
#pragma unroll
                        for (int j = 0; j < 16 / (int)sizeof(T); ++j) x[k * (QN / R::kPasses) + s][i + j] = (float)v[j];
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < QN; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[s][i]) & 0x7fffffffu);
            top = max(top, __float_as_uint(swap32(__uint_as_float(top))));
            bad = top >= 0x7f800000u;
            const int e = P == 2 && !bad ? max((int)(top >> 23), 1) - 127 - 14 : 0;
            if constexpr (P == 2) cs = ldexpf(a.scale2, e);
            cs = finite_factor(cs);
#pragma unroll
            for (int s = 0; s < QN; ++s)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y = bad ? 0.0f : P == 2 ? ldexpf(x[s][i], -e) : x[s][i];
                    q[0][s][i] = (_Float16)y;
                    if constexpr (P == 2) q[1][s][i] = (_Float16)(y - (float)q[0][s][i]);
                }
        }
        typedef float f16v __attribute__((ext_vector_type(16)));
        f16v o[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = (f16v){};
        // p = 2^(s cs + c2), c2 = kBias - m cs rounded (infinite while m is -infinity); where that would cost
        // the last bits of a score (far) the difference to m is taken first
        float m = -INFINITY, c2 = INFINITY, l = 0.0f;
        uint32_t far = 0;   // uniform
        const uint32_t kat = lane * 16u;
        uint32_t vat[2];   // of even and odd blocks of dims: the slots are permuted by (dim / 8) % 8
#pragma unroll
        for (int d = 0; d < 2; ++d) vat[d] = (((col >> 3) * 8u + ((col & 7u) ^ ((4u * d + (col >> 3)) & 7u))) + 32u * h) * 16u;
        uint32_t b = 0;
        if (p0 < p1) {
            store(0);
            load(min(p0 + TP, last_tile));
        }
        for (uint32_t p = p0; p < p1; p += TP, b ^= 1u) {
            __syncthreads();   // this tile is there, the other buffer has been read
            if (p + TP < p1) {
                store(b ^ 1u);
                // past the end the last tile again: under a condition the compiler would wait for these loads at once
                load(min(p + 2 * TP, last_tile));
            }
            const uint32_t first = p + 32u * phase;   // NB blocks of 32 positions
            if (first >= wave_hi) continue;
            const uint8_t *kt = smem + b * 2 * kTile + phase * (QN * 1024u), *vt = smem + b * 2 * kTile + kTile + phase * (2 * ND * 1024u);
            f16v s[NB];
            fh8 k[NB][QN];
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int t = 0; t < QN; ++t) k[n][t] = *(const fh8 *)(kt + kat + (n * QN + t) * 1024u);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                s[n] = (f16v){};
                if constexpr (P == 2)   // the small parts first
#pragma unroll
                    for (int t = 0; t < QN; ++t) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[n][t], q[1][t], s[n], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < QN; ++t) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[n][t], q[0][t], s[n], 0, 0, 0);
            }
            // half the operands are requested together, the others one by one behind the products: left to
            // itself the compiler waits for every two before it asks for the next
            if constexpr (P == 1) {
                constexpr int kAhead = NB * QN / 2;
                __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
                for (int t = 0; t < NB * QN - kAhead; ++t) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
            }
            if (first + 32u * NB > min(wave_lo, p1)) {   // some column does not see all, or positions beyond the part are not its own
                const uint32_t below = min(vis, p1);
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int v = 0; v < 16; ++v) s[n][v] = first + 32 * n + 8 * (v >> 2) + 4 * h + (v & 3) < below ? s[n][v] : -INFINITY;
            }
            float top[2] = {s[0][0], s[0][1]};
#pragma unroll
            for (int x = 2; x < 16 * NB; ++x) top[x & 1] = fmaxf(top[x & 1], s[x >> 4][x & 15]);
            float bm = fmaxf(top[0], top[1]);
            bm = fmaxf(bm, swap32(bm));
            // far scores always enter: c2 may be rounded by more than the slack, and p would leave binary16's range
            if (__builtin_amdgcn_readfirstlane(far | (__any(fmaf(bm, cs, c2) > kBias + kSlack) ? 1u : 0u))) {
                const float now = fmaxf(m, bm), cn = now == -INFINITY ? INFINITY : fmaf(-now, cs, kBias);
                float f;
                if (__builtin_amdgcn_readfirstlane(far | (__any(fabsf(cn) > 4194304.0f && now != -INFINITY) ? 1u : 0u))) {   // cn itself may be infinite
                    // from c2 as it was rounded to the difference: all but kBias of it cancels in one FMA
                    // (kBias - c2 by itself loses 1/4 where c2 is below kBias - 2^22)
                    const float r = far ? 0.0f : fmaf(-m, cs, -c2) + kBias;
                    f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(fmaf(m - now, cs, r));
                    far = 1;
                } else {
                    f = cn == c2 ? 1.0f : __builtin_amdgcn_exp2f(cn - c2);
                }
                m = now;
                c2 = cn;
                l *= f;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int v = 0; v < 16; ++v) o[d][v] *= f;
            }
            float off = m == -INFINITY ? 0.0f : c2;
            if (__builtin_amdgcn_readfirstlane(far)) {
                const float m0 = m == -INFINITY ? 0.0f : m;
                off = kBias;
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int v = 0; v < 16; ++v) s[n][v] -= m0;
            }
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int t = 0; t < 2 * NB; ++t) {
                fh8 ph, pl;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(s[t >> 1][8 * (t & 1) + e], cs, off));
                    ph[e] = (_Float16)x;
                    if constexpr (P == 2) {
                        pl[e] = (_Float16)(x - (float)ph[e]);
                        sum[e & 1] += x;
                    }
                }
                if constexpr (P == 1) {   // of P as rounded: both sums see the same weights
                    const jh2 one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
                    for (int e = 0; e < 8; e += 2) sum[(e >> 1) & 1] = __builtin_amdgcn_fdot2(jh2{ph[e], ph[e + 1]}, one, sum[(e >> 1) & 1], false);
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const fh8 v = *(const fh8 *)(vt + vat[d & 1] + (t * ND + d) * 1024u);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph, o[d], 0, 0, 0);
                    if constexpr (P == 2) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl, o[d], 0, 0, 0);
                }
            }
            l += sum[0] + sum[1];
        }
        l += swap32(l);
        // from here on the weights are multiples of 2^(m cs - less), as the roundings have left them: kBias - c2 for m would
        // be off by up to 2^-21 (1/4 near 2^22), and so would all weights of a phase or part, against those of the others
        float less = far ? kBias : 0.0f;
        if (!far) {
            m = m == -INFINITY ? m : -c2;
            cs = 1.0f;
        }
        const bool odd = p0 < p1 && __syncthreads_or(worst > 140u);
        if constexpr (PH == 2) {
            // the second phase's state goes through the first tile, its m, factor, less and l through where its rows were
            float *const state = (float *)(smem + (wave & 1u) * kTile) + lane;
            float *const sums = (float *)(smem + 2 * kTile + (2u + (wave & 1u)) * (kTile / 2)) + lane;
            if (phase) {
                sums[0] = m;
                sums[64] = cs;
                sums[128] = l;
                sums[192] = less;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int v = 0; v < 16; ++v) state[(16 * d + v) * 64] = o[d][v];
            }
            __syncthreads();
            if (!phase) {
                const float m2 = sums[0], cs2 = sums[64];
                const double e1 = (double)m * (double)cs - less, e2 = (double)m2 * (double)cs2 - sums[192];
                const float f1 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((float)(e1 - fmax(e1, e2)));
                const float f2 = m2 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((float)(e2 - fmax(e1, e2)));
                l = l * f1 + sums[128] * f2;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int v = 0; v < 16; ++v) o[d][v] = o[d][v] * f1 + state[(16 * d + v) * 64] * f2;
                if (e2 > e1) {
                    m = m2;
                    cs = cs2;
                    less = sums[192];
                }
            }
        }
        const float nan = __uint_as_float(0x7fc00000u);
        if (odd && !idle) {
            const Nans<D> at = all_nans<D>(ks, vs, srow, p0, wave_hi);
            if (at.k < vis) l = nan;
#pragma unroll
            for (int d = 0; d < ND; ++d)
                if (at.v[d] < vis)
#pragma unroll
                    for (int v = 0; v < 16; ++v) o[d][v] = nan;
        }
        __syncthreads();   // the tiles have been read: the results pass through them, or the next columns' do
        const bool there = phase == 0 && c0 + col < columns;
        if (bad && vis) l = nan;
        const Fp4Args &z = late_args<Fp4Args>();
        if (SPLIT && w.parts > 1) {
            const size_t at = ((size_t)w.slot * z.kv_heads + kvh) * z.cols + (c - w.c0);
            float *to = z.part + at * D;
            if (there) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *(jf4 *)(to + 32 * d + 8 * j + 4 * h) = jf4{o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]};
            }
            if (there && h == 0) *(ff4 *)(z.part_ml + 4 * at) = ff4{m, cs, l, less};
        } else {
            typedef Rows<T, D, TP> R;
            const float inv = vis ? 1.0f / l : 0.0f;
            uint8_t *const stage = smem + 2 * kTile + wave * (32u * R::kBytes);
            const uint32_t lane = fresh_thread() & 63u, col = lane & 31u, h = lane >> 5, piece = lane % R::kPieces, r0 = lane / R::kPieces;
#pragma unroll
            for (int k = 0; k < R::kPasses; ++k) {
                constexpr int N = ND / R::kPasses;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (int d = 0; d < N; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        typedef T t4 __attribute__((ext_vector_type(4)));
                        t4 y;
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[i] = vis ? (T)(o[k * N + d][4 * j + i] * inv) : (T)0.0f;
                        const uint32_t at = (32u * d + 8u * j + 4u * h) * sizeof(T);
                        *(t4 *)(stage + R::place(col, at / 16u) + at % 16u) = y;
                    }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (int i = 0; i < R::kTurns; ++i) {
                    const uint32_t r = r0 + i * (64u / R::kPieces);
                    T *to = (T *)z.out + (size_t)__shfl(qat, (int)r) * D + k * R::kDims + piece * (16 / sizeof(T));
                    const ju4 y = *(const ju4 *)(stage + R::place(r, piece));
                    if (phase == 0 && c0 + r < columns) *(ju4 *)to = y;
                }
            }
        }
        if (SPLIT && there && w.slot == w.first_slot && kvh == 0 && h == 0) {
            uint32_t *to = z.meta + 2 * ((size_t)w.s.row0 * z.G + c);
            to[0] = w.first_slot;
            to[1] = w.parts | (vis ? 0u : 1u << 23) | (c - w.c0) << 24;
        }
    }
}

template <typename K> int launch(janus_ctx *ctx, K kernel, dim3 grid, dim3 block, uint32_t lds, const Fp4Args &a) {
    hipLaunchKernelGGL(kernel, grid, block, lds, ctx->stream, a);
    JANUS_LAUNCH_CHECK(ctx);
    return JANUS_OK;
}

// How a launch is cut up. cols columns a workgroup, of per_cu on a CU; many columns are split from `fewest` steps on.
void plan(janus_ctx *ctx, Fp4Args &a, uint32_t cols, uint32_t hw, uint32_t ph, uint32_t step, uint32_t per_cu, uint32_t fewest, uint32_t max_len) {
    a.cols = cols;
    a.hw = hw;
    a.ph = ph;
    a.step = step;
    a.head_groups = a.kv_heads / hw;
    a.least = 2;
    a.target = 0;
    // every tile of every sequence, one more where rows do not fill the last
    const uint64_t tiles = (uint64_t)a.rows * a.G / cols + a.nseq, mean = (a.rows + a.nseq - 1) / a.nseq;
    a.shares = (uint32_t)tiles;   // * head_groups below 2^21 + 2^22, up to 512 lanes each
    a.slots = 0;
    const uint64_t busy = std::max<uint64_t>(1, std::min<uint64_t>(tiles, ((uint64_t)a.rows * a.G + cols - 1) / cols + a.nseq - 1));
    const uint64_t at_once = std::max<uint64_t>(1, (uint64_t)ctx->num_cus * per_cu / a.head_groups);
    const bool counts = tiles * (std::min(a.max_seq, a.cache_rows) / step + 1) < (1ull << 31);   // units of all tiles
    // A split costs a second launch and a search over the sequences for every share; without one a
    // workgroup takes 0.7 to 1.5 us for 32 positions. Where both were measured (8 KV heads of 128
    // dims, up to 1000 sequences of up to 4000 positions) they meet at 10 steps and 20 more for
    // as many workgroups as run at once: decode steps of 64 sequences of up to 1600 positions take
    // 31 us split and 77 whole, 300 of up to 400 take 45 and 37, 300 of up to 1600 83 and 114.
    // Many columns: whole tiles leave CUs idle where there are few, but shares of equal length count
    // positions that early rows of a prompt do not see: 512 rows behind 1500 positions 41 us split and
    // 50 whole, 1024 behind 1024 63 and 51, and 4 x 512 behind 2000 109 and 80.
    const uint64_t steps = max_len / step;
    const bool split = cols <= 16 ? steps * at_once > 10 * at_once + 20 * busy && busy < 4 * at_once
                                  : steps > fewest && 2 * busy <= at_once && 3 * mean <= max_len;
    if (counts && split) {
        // at most 128 parts of a tile in the mean, which the join's 16 wavefronts read in one go: a sequence of 16000
        // positions in 250 parts 21 us, in 125 18 to 19. The lengths are on the device: a long sequence beside short ones has
        // more parts, and a join for the mean (that one and one of a single position 22 us, and 63 of 20 positions 64)
        a.shares = a.target = (uint32_t)std::min<uint64_t>(at_once, 128 * busy);
        a.slots = (uint32_t)(a.shares + tiles);
        a.mean_parts = (uint32_t)std::min<uint64_t>(a.shares / busy, steps / a.least) + 1;
    }
}

int reserve(janus_ctx *ctx, Fp4Args &a, uint32_t D) {
    if (!a.target) return JANUS_OK;
    const size_t cells = (size_t)a.slots * a.kv_heads * a.cols;
    const size_t meta = ((size_t)a.rows * a.G * 8 + 255) / 256 * 256;
    if (int e = ensure_attn_ws(ctx, meta + cells * (D + 4) * 4)) return e;
    a.meta = (uint32_t *)ctx->attn_ws;
    a.part = (float *)((char *)ctx->attn_ws + meta);
    a.part_ml = a.part + cells * D;
    return JANUS_OK;
}

// KV heads of a few-column workgroup.
uint32_t few_heads(uint32_t kv_heads, uint32_t waves) {
    while (kv_heads % waves) waves /= 2;
    return waves;
}

template <typename T, int D, int NW, int PER> int launch_few(janus_ctx *ctx, Fp4Args &a, uint32_t max_len) {
    const uint32_t hw = few_heads(a.kv_heads, NW), ph = NW / hw;
    // two tiles, or the phases' results: 64 KB at most
    const uint32_t lds = std::max<uint32_t>(Tile<D, NW>::kLds, (ph - 1) * hw * (D / 4 + 2) * 256u);
    plan(ctx, a, 16, hw, ph, 32 * ph, std::min<uint32_t>(PER * 4 / NW, 160 * 1024 / lds), 0, max_len);
    if (int e = reserve(ctx, a, D)) return e;
    const dim3 grid((a.shares + 7) / 8 * 8 * a.head_groups), block(NW * 64);
    if (a.target) return launch(ctx, fp4_attn_kernel<T, D, NW, PER, true>, grid, block, lds, a);
    return launch(ctx, fp4_attn_kernel<T, D, NW, PER, false>, grid, block, lds, a);
}

template <typename T, int D, int PH> int launch_wide(janus_ctx *ctx, Fp4Args &a, uint32_t max_len) {
    constexpr int TP = PH == 1 && D == 128 && sizeof(T) == 4 ? 32 : 64;
    // a step of two-part rows takes twice as long; tiles of 128 such columns are more than the CUs (launch_dim) and stay whole
    constexpr bool kWhole = PH == 1 && sizeof(T) == 4;
    plan(ctx, a, 128 / PH, 1, 1, 64, 2, kWhole ? 0xffffffffu : sizeof(T) == 4 ? 10 : 16, max_len);
    if (int e = reserve(ctx, a, D)) return e;
    const dim3 grid(a.shares * a.kv_heads), block(256);
    if constexpr (!kWhole)
        if (a.target) return launch(ctx, fp4_wide_kernel<T, D, TP, PH, true>, grid, block, 4 * TP * D * 2, a);
    return launch(ctx, fp4_wide_kernel<T, D, TP, PH, false>, grid, block, 4 * TP * D * 2, a);
}

template <typename T, int D> int launch_dim(janus_ctx *ctx, Fp4Args &a, uint32_t max_len) {
    const uint64_t columns = (uint64_t)((a.rows + a.nseq - 1) / a.nseq) * a.G;   // of a sequence and KV head, in the mean
    // what fits the registers: q and O of 16 columns in 128 of them (two workgroups of eight wavefronts on a CU),
    // with two-part q of 128 dims in 160 (three of four wavefronts)
    constexpr bool kTwo = sizeof(T) == 4 && D == 128;
    constexpr int NW = kTwo ? 4 : 8, PER = kTwo ? 3 : 4;
    // A few-column workgroup of one or two KV heads (hw: the largest power of two in their number, up to NW) has many
    // phases, 64 to 256 positions at a time where the other kernel takes 64: while all its tiles run at once that is the shorter chain, though each reads K and V (16/1/128, 64 x 3 rows
    // behind up to 2000: 19 and 27 us, binary32 22 and 31; 40 x 3 behind 600 12 and 17, 12 and 22). Long contexts of
    // binary16 rows are bound by those reads (64 x 3 behind up to 7800 43 and 36, binary32 44 and 44; 300 x 3 behind 1000
    // 34 and 30), and with eight heads a step is 32 positions (32/8/128, 40 x 8 behind 600: 41 and 20). Three, five, six and
    // ten KV heads go the same way: 12 x 40 columns behind 600 12 and 19 at 24/3/128, 13 and 19 at 40/5/128, 15 and 19 at
    // 24/6/128, 16 and 20 at 40/10/128 (binary32 13 and 24, 13 and 24, 17 and 24, 18 and 24); 60 columns of ten heads behind
    // 2000 lose (4 sequences 31 and 26, 12 33 and 34, binary32 52 and 40).
    const uint32_t hw = few_heads(a.kv_heads, NW);
    const uint64_t tiles = ((uint64_t)a.rows * a.G + 15) / 16 + a.nseq - 1;
    const bool many_phases = hw <= 2 && tiles * (a.kv_heads / hw) <= (uint64_t)ctx->num_cus * (PER * 4 / NW) &&
                             (sizeof(T) == 4 || max_len <= 2048);
    // Pairs of wavefronts also where tiles of 128 columns would leave a place of every CU free: half the columns and
    // half the work of each step. One prompt of 1000 rows at 32/8/128: 31 and 27 us, binary32 51 and 37; of 2000 at
    // 16/1/128 51 and 42, 86 and 58. Short binary16 rows gain nothing from there being more of them (16 prompts of 120
    // at 16/1/128: 11 and 13 us, 4 of 500 19 and 20, one of 300 at 32/8/128 14 and 13). Where the steps of two-part rows
    // of 128 dims are long, and those of binary16 ones of 64 short, also for both places of every CU (1500 rows at
    // 32/8/128 binary32 72 and 61, at 24/8/64 binary16 29 and 26; 2000 binary16 ones at 32/8/128 59 and 66, 8 x 250
    // binary32 ones at 24/8/64 17 and 22).
    const uint64_t wide = (((uint64_t)a.rows * a.G + 127) / 128 + a.nseq - 1) * a.kv_heads, cus = (uint64_t)ctx->num_cus;
    const bool pairs = columns <= 64 || 2 * wide <= cus || (wide <= (kTwo || (sizeof(T) == 2 && D == 64) ? 2 * cus : cus) &&
                                                                 (sizeof(T) == 4 || a.rows / a.nseq >= 512));
    int e;
    if (columns <= 16 || (columns <= 64 && many_phases)) e = launch_few<T, D, NW, PER>(ctx, a, max_len);
    else if (pairs) e = launch_wide<T, D, 2>(ctx, a, max_len);
    else e = launch_wide<T, D, 1>(ctx, a, max_len);
    if (e || !a.target) return e;
    const uint32_t units = a.rows * a.heads;
    if (a.mean_parts <= 8) hipLaunchKernelGGL((fp4_join_kernel<T, D, 1>), dim3((units + 3) / 4), dim3(256), 0, ctx->stream, a);
    else if (a.mean_parts <= 32) hipLaunchKernelGGL((fp4_join_kernel<T, D, 4>), dim3(units), dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL((fp4_join_kernel<T, D, 16>), dim3(units), dim3(1024), 0, ctx->stream, a);
    JANUS_LAUNCH_CHECK(ctx);
    return JANUS_OK;
}

}  // namespace

int fp4_attention_launch(janus_ctx *ctx, const void *q, int q_dt, const uint8_t *kc, const uint8_t *ks,
                         const uint8_t *vc, const uint8_t *vs, void *out, uint32_t rows, uint32_t nseq, uint32_t heads,
                         uint32_t kv_heads, uint32_t hd, uint32_t cache_rows, uint32_t max_seq, const int32_t *q_start,
                         const int32_t *row_base, const int32_t *seq_lens, uint32_t max_len, float scale) {
    Fp4Args a{};
    a.q = q;
    a.kc = kc;
    a.ks = ks;
    a.vc = vc;
    a.vs = vs;
    a.out = out;
    a.q_start = q_start;
    a.row_base = row_base;
    a.seq_lens = seq_lens;
    a.rows = rows;
    a.nseq = nseq;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.G = heads / kv_heads;
    a.cache_rows = cache_rows;
    a.max_seq = max_seq;
    a.scale2 = scale * 1.44269504088896340736f;
    if (q_dt == JANUS_DT_F16) return hd == 128 ? launch_dim<_Float16, 128>(ctx, a, max_len) : launch_dim<_Float16, 64>(ctx, a, max_len);
    return hd == 128 ? launch_dim<float, 128>(ctx, a, max_len) : launch_dim<float, 64>(ctx, a, max_len);
}

}  // namespace janus
