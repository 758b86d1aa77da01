// attend.hpp - attention over two ranges of keys, in the caches' own type
// (f32, f16, bf16): rows that see a sliding window and the first positions of
// their sequence, and rows of a batch of sequences that share one prefix.
//
// Row i of sequence b sees all of the shared range and, of the sequence's own
// range, the positions j <= p(i) with j < n_sink, window == 0 or j > p(i) - window:
//   s_j = <q, k_j> / sqrt(D),  o = sum_j e^(s_j - max) v_j / sum_j e^(s_j - max)
// Scores, exponents, sums and the output's accumulation are f32; the output is
// rounded once to the caches' type. A row that sees nothing is 0.
//
// One pass over the keys with the running maximum and sum. Every kernel works
// on transposed products: S^T = K Q^T puts a query row in a lane (the row's
// maximum and sum are in-lane operations plus one or two exchanges), and the
// accumulator layout of S^T is, up to the order of the keys, the operand layout
// of P^T in O^T = V^T P^T. So the weights go from the first product to the
// second in registers, and only V's operand is read in that order of keys.
// 16-bit weights go into the second product in the caches' type. Up to 32 rows of a
// sequence (positions x heads of a group; 16 with heads of 256) as two parts,
// rounded and rest: bound by memory, the product of the rest is free (one row,
// 32784 bf16 keys: 41.0 and 41.4 us, error 2.5e-3 and 1.6e-3). The prefix's blocks,
// over the rows of all such sequences, keep both parts too, so that a row is as
// exact in a large batch as alone (bf16, a call of 64 sequences behind 8192 53.7 us
// rounded and 54.6 so, error 2.3e-3 and 1.7e-3; where the prefix outweighs the tails,
// 64 behind 30000: 83 and 95 us). Sequences of more rows are bound by the products:
// there rounded, half a step each against values that are themselves rounded so.
// The sum takes them rounded too, so that equal values stay what they are (8192
// rows: 492 us with the sum before rounding, 490 so).
//
// A block takes one kv head, a tile of rows (all query heads of the group x
// positions, heads fastest) and a run of key tiles. Where runs are cut or a
// prefix is joined to tails, blocks leave (maximum, sum, accumulator) in f32
// and k_join puts them together.
#pragma once

#include <type_traits>

#include "device.hpp"
#include "internal.hpp"

namespace aotk {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
// 16, 8 and 4 bytes at any element's alignment
typedef uint32_t u32x4e __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2e __attribute__((ext_vector_type(2), aligned(2)));

constexpr float NEG_INF = -__builtin_inff();
// The running maximum moves only when a row's grows by more than 2^8: until
// then weights are up to 2^8 times too large, and the accumulator is not rescaled.
constexpr float RESCALE = 8.0f;
// Weights are kept 2^LIFT times as large. f16: 2^6 (2^14 at most), since below
// 2^-14 an f16 loses bits, and a long row may have many weights that small beside
// one large; its values are too small to overflow. The other types hold values as
// large as f32 itself: at 2^-8 their weights are at most 1, and the sums overflow
// where those of the formula do (values below 2^-118 may lose bits). bf16 takes the 2^-8 in the exponent; there it
// would cost f32 weights two bits, which are multiplied by it instead.
template <int KIND>
constexpr float LIFT = KIND == AOTK_F16 ? 6.0f : (KIND == AOTK_BF16 ? -RESCALE : 0.0f);
template <int KIND>
__device__ __forceinline__ float att_weight(float score, float scale_log2, float base) {
    const float w = __builtin_amdgcn_exp2f(fmaf(score, scale_log2, -base));
    return KIND == AOTK_F32 ? w * 0x1p-8f : w;
}

template <int KIND>
struct AttElem {
    typedef uint16_t elem;
    static __device__ __forceinline__ bool finite(uint32_t x) {
        return KIND == AOTK_F16 ? (x & 0x7C00u) != 0x7C00u : (x & 0x7F80u) != 0x7F80u;
    }
    static __device__ __forceinline__ float up(uint32_t x) { return KIND == AOTK_F16 ? f16_to_f32(x) : bf16_to_f32(x & 0xFFFFu); }
    static __device__ __forceinline__ uint32_t pair(float a, float b) {  // to nearest even
        if constexpr (KIND == AOTK_F16) {
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            return __builtin_bit_cast(uint32_t, h2{(_Float16)a, (_Float16)b});
        } else {
            typedef __bf16 b2 __attribute__((ext_vector_type(2)));
            return __builtin_bit_cast(uint32_t, b2{(__bf16)a, (__bf16)b});
        }
    }
    // both values of a pair
    static __device__ __forceinline__ float first(uint32_t x) {
        if constexpr (KIND == AOTK_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)x);
        else return __uint_as_float(x << 16);
    }
    static __device__ __forceinline__ float second(uint32_t x) {
        if constexpr (KIND == AOTK_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(x >> 16));
        else return __uint_as_float(x & 0xFFFF0000u);
    }
    static __device__ __forceinline__ float add_pair(uint32_t x, float sum) {  // sum + first + second, one instruction
        if constexpr (KIND == AOTK_F16) {
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, x), h2{(_Float16)1, (_Float16)1}, sum, false);
        } else {
            typedef __bf16 b2 __attribute__((ext_vector_type(2)));
            return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, x), __builtin_bit_cast(b2, 0x3F803F80u), sum, false);
        }
    }
    static __device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
        if constexpr (KIND == AOTK_F16)
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
        if constexpr (KIND == AOTK_F16)
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
    }
};
template <>
struct AttElem<AOTK_F32> {
    typedef float elem;
    static __device__ __forceinline__ bool finite(uint32_t x) { return (x & 0x7F800000u) != 0x7F800000u; }
    static __device__ __forceinline__ float up(float x) { return x; }
};

// Four contiguous outputs from dimension d on, rounded to the caches' type.
template <int KIND>
__device__ __forceinline__ void store4(void *out, size_t at, float a, float b, float c, float d) {
    if constexpr (KIND == AOTK_F32) *(u32x4e *)((float *)out + at) = u32x4{__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d)};
    else *(u32x2e *)((uint16_t *)out + at) = u32x2{AttElem<KIND>::pair(a, b), AttElem<KIND>::pair(c, d)};
}

// A block's part of a launch: keys, sequence, rows, run of key tiles.
struct AttJob {
    const void *ka, *va, *k, *v;  // ranges A and B, of the sequence and kv head
    uint64_t window, n_sink;
    uint32_t kvh, group, causal;
    uint32_t row0;
    uint64_t part0;      // first row's place among partial results
    uint32_t r0, nr;     // rows r0.. of the sequence's rows x group, nr of them
    int64_t pmin, pmax;  // positions of the first and the last of them
    uint64_t na, b0, nb; // keys of A; first and number of keys of B
    uint32_t ta, t0, t1; // tiles of A; the run
    bool direct;         // the only results of these rows: to the output
    bool any_a;
    // element offset of row rr in q and out, and its place among partial results
    __device__ __forceinline__ size_t at(const AttendLaunch &a, uint32_t rr, int D) const {
        return ((size_t)(row0 + rr / group) * a.n_head + kvh * group + rr % group) * D;
    }
    __device__ __forceinline__ size_t slot(const AttendLaunch &a, uint32_t rr) const {
        return (part0 + rr / group) * a.n_head + kvh * group + rr % group;
    }
    __device__ __forceinline__ int rel(uint32_t rr) const { return causal ? (int)(rr / group - r0 / group) : 0; }
    __device__ __forceinline__ bool sees_any(uint32_t rr) const { return any_a || pmin + rel(rr) >= 0; }
};

template <typename E, int D, int ROWS, int NK>
__device__ __forceinline__ AttJob att_job(const AttendLaunch &a, bool prefix) {
    AttJob w;
    // (by index: a choice between two members of the arguments would have
    // them copied to scratch memory first)
    const AttendView &r = a.range[prefix ? 1 : 0];
    uint32_t item = blockIdx.x - r.block0, si = r.seq0;
    if (!prefix && a.n_seq > 1) {  // the last sequence whose first block is not past this one
        const int lane = threadIdx.x & 63;
        const bool le = lane < (int)a.n_seq && a.seq[lane].block0 <= item;
        si = (uint32_t)__builtin_amdgcn_readfirstlane(__popcll(__ballot(le)) - 1);
    }
    const AttendPlace &s = a.seq[si];
    item -= s.block0;
    const uint32_t run = r.run;
    w.window = r.window;
    w.n_sink = r.n_sink;
    w.causal = r.causal;
    w.kvh = item % a.n_kv_head;
    item /= a.n_kv_head;
    w.group = a.n_head / a.n_kv_head;
    w.row0 = s.row0;
    const uint32_t chunk = item % s.chunks;
    w.part0 = s.part0 + (uint64_t)chunk * s.rows;
    const uint32_t tile = item / s.chunks, all = s.rows * w.group, row_tiles = (all + ROWS - 1) / ROWS;
    // the last rows see most: they start first
    w.r0 = (row_tiles - 1 - tile) * ROWS;
    w.nr = all - w.r0 < ROWS ? all - w.r0 : ROWS;
    const int64_t first = (int64_t)s.len - s.rows;
    w.pmin = w.causal ? first + w.r0 / w.group : (int64_t)s.len - 1;
    w.pmax = w.causal ? first + (w.r0 + w.nr - 1) / w.group : (int64_t)s.len - 1;
    const AttendSpan sp = attend_span(r.na, w.window, w.n_sink, w.pmin, w.pmax);
    w.na = sp.na;
    w.b0 = sp.b0;
    w.nb = sp.nb;
    w.ta = (uint32_t)((w.na + NK - 1) / NK);
    const uint32_t tiles = w.ta + (uint32_t)((w.nb + NK - 1) / NK);
    const uint64_t c0 = (uint64_t)chunk * run;
    w.t0 = c0 < tiles ? (uint32_t)c0 : tiles;
    w.t1 = c0 + run < tiles ? (uint32_t)(c0 + run) : tiles;
    w.direct = s.chunks == 1 && !a.joined;
    w.any_a = r.na > 0;
    const size_t kv = (size_t)a.n_kv_head * D;
    const size_t own = s.cache * kv + w.kvh * D;
    w.k = (const E *)r.k + own;
    w.v = (const E *)r.v + own;
    const size_t at_a = r.na ? w.kvh * D : own;  // the prefix, or the sequence's first positions
    w.ka = (const E *)r.ka + at_a;
    w.va = (const E *)r.va + at_a;
    return w;
}

// A key tile: its rows in memory, how many keys it has, where it is.
template <typename E>
struct AttTile {
    const E *k, *v;
    uint32_t n;
    int64_t j0;
    bool ragged;  // rows of the block differ in what they see of it
};

template <typename E, int NK>
__device__ __forceinline__ AttTile<E> att_tile(const AttJob &w, size_t kv, uint32_t t) {
    AttTile<E> x;
    if (t < w.ta) {
        const uint64_t j = (uint64_t)t * NK;
        x.k = (const E *)w.ka + j * kv;
        x.v = (const E *)w.va + j * kv;
        x.n = w.na - j < NK ? (uint32_t)(w.na - j) : NK;
        x.j0 = 0;
        x.ragged = false;
    } else {
        const uint64_t j = (uint64_t)(t - w.ta) * NK;
        x.k = (const E *)w.k + (w.b0 + j) * kv;
        x.v = (const E *)w.v + (w.b0 + j) * kv;
        x.n = w.nb - j < NK ? (uint32_t)(w.nb - j) : NK;
        x.j0 = (int64_t)(w.b0 + j);
        x.ragged = w.causal && !(x.j0 + x.n - 1 <= w.pmin && (w.window == 0 || x.j0 > w.pmax - (int64_t)w.window ||
                                                             x.j0 + x.n <= (int64_t)w.n_sink));
    }
    return x;
}

// Keys of a tile of n that a row sees: `c` the key's number in the tile, `rel`
// the row's position behind the block's first. What is far outside the tile is
// clipped, beyond any `rel`. Without branches, for selects: as conditions with
// short cuts the 16 to 32 tests of a lane become as many jumps.
struct AttSees {
    int hi, lo, sink;
    template <typename E>
    __device__ __forceinline__ AttSees(const AttJob &w, const AttTile<E> &x, int rel) {
        constexpr int64_t FAR = 1 << 30;
        auto clip = [](int64_t y) { return (int)(y < -FAR ? -FAR : (y > FAR ? FAR : y)); };
        hi = min(x.ragged ? clip(w.pmin - x.j0) + rel : (int)x.n - 1, (int)x.n - 1);
        lo = x.ragged && w.window ? clip(w.pmin - (int64_t)w.window - x.j0) + rel : -1;
        sink = clip((int64_t)w.n_sink - x.j0);
    }
    __device__ __forceinline__ bool operator()(int c) const { return (c <= hi) & ((c > lo) | (c < sink)); }
};

// Maximum and sum with the lane 16 or 32 away: swaps of 16-lane rows and of
// halves in the registers, not through LDS.
__device__ __forceinline__ f32x2 swap16(float x) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f32x2{__uint_as_float(r[0]), __uint_as_float(r[1])};
}
__device__ __forceinline__ f32x2 swap32(float x) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f32x2{__uint_as_float(r[0]), __uint_as_float(r[1])};
}
__device__ __forceinline__ float max32(float x) {
    const f32x2 r = swap32(x);
    return fmaxf(r[0], r[1]);
}
__device__ __forceinline__ float max16(float x) {
    const f32x2 r = swap16(x);
    return fmaxf(r[0], r[1]);
}
__device__ __forceinline__ float sum32(float x) {
    const f32x2 r = swap32(x);
    return r[0] + r[1];
}
__device__ __forceinline__ float sum16(float x) {
    const f32x2 r = swap16(x);
    return r[0] + r[1];
}

// New running maximum of a row (in units of the exponent): the base to
// subtract, and the factor for what was summed so far.
__device__ __forceinline__ float att_base(float mc) { return mc == NEG_INF ? 0.0f : mc; }
__device__ __forceinline__ float att_shift(float from, float to) { return from == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(from - to); }

// --------------------------------------------------------------- few rows
// Up to 16 * RB rows against a long run of keys: bound by memory. Each of NW
// waves takes every NW-th tile of the run for itself and reads K and V straight into
// the operand registers, 16 bytes per lane and load; the next tile's K is
// requested as soon as the scores are formed, its V after the second product.
// V arrives as a lane's 8 keys x 8 dimensions and is transposed there by byte
// permutes. The waves' results meet in LDS at the end.
// One bf16 row, 32 heads over 8 of 128, 32784 keys: 134 MB in 24.6 us, 5.5 TB/s (a
// large copy reaches 6.2). One f32 row of 1028 keys: 9.4 us, the latency of one
// tile from the arguments to the result, of which the memory takes 2.
template <int KIND, int D>
struct NarrowShape {
    static constexpr bool F32 = KIND == AOTK_F32;
    static constexpr int NK = F32 ? 16 : 32;          // keys of a tile
    static constexpr int KR = D / 16;                 // 16-byte loads of K per lane
    static constexpr int VL = F32 ? D / 64 : (D == 256 ? 2 : 1);  // loads per key of V
    static constexpr int VK = F32 ? 4 : 8;            // keys of V per lane
    static constexpr int CW = F32 ? 4 : (D == 64 ? 4 : 8);  // dimensions per load of V
    static constexpr int QR = F32 ? D / 16 : D / 32;  // 16-byte registers of q
    static constexpr int NA = D / 16;                 // accumulators of 16 dimensions x 16 rows
    template <int NW, int RB>
    static constexpr size_t lds_bytes() { return (size_t)NW * 16 * RB * ((D + 4) * 4 + 8); }
    // dimension of accumulator c, row m of its 16
    static __device__ __forceinline__ int dim(int c, int m) { return c / CW * (16 * CW) + m * CW + c % CW; }
};

template <int KIND, int D, int NW, int RB>
__device__ __forceinline__ void attend_narrow(const AttendLaunch &a, bool prefix, uint8_t *lds) {
    typedef NarrowShape<KIND, D> S;
    typedef typename AttElem<KIND>::elem E;
    constexpr int NK = S::NK, ROWS = 16 * RB;
    constexpr bool F32 = S::F32;
    const AttJob w = att_job<E, D, ROWS, NK>(a, prefix);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
    const size_t kv = (size_t)a.n_kv_head * D;
    const uint32_t kvb = a.n_kv_head * (uint32_t)(D * sizeof(E));  // bytes between keys

    u32x4 q[RB][S::QR];
    int rel[RB];  // the lane's row's position behind the block's first
#pragma unroll
    for (int b = 0; b < RB; b++) {
        const uint32_t rr = w.r0 + b * 16 + n;
        rel[b] = 0;
#pragma unroll
        for (int u = 0; u < S::QR; u++) q[b][u] = u32x4{0, 0, 0, 0};
        if ((uint32_t)(b * 16 + n) < w.nr) {
            rel[b] = w.rel(rr);
            const E *src = (const E *)a.q + w.at(a, rr, D);
#pragma unroll
            for (int u = 0; u < S::QR; u++) q[b][u] = *(const u32x4e *)(src + (F32 ? 16 * u + 4 * g : 32 * u + 8 * g));
        }
    }
    f32x4 acc[RB][S::NA];
    float mc[RB], sum[RB];
#pragma unroll
    for (int b = 0; b < RB; b++) {
        mc[b] = NEG_INF;
        sum[b] = 0.0f;
#pragma unroll
        for (int c = 0; c < S::NA; c++) acc[b][c] = f32x4{0, 0, 0, 0};
    }

    u32x4 k[S::KR], v[S::VK * S::VL];
    // keys past the tile's end read its last key; their scores are masked and
    // their values are zeroed below
    auto v_key = [&](int j) { return F32 ? 4 * g + j : (j < 4 ? 4 * g + j : 16 + 4 * g + j - 4); };
    auto load_k = [&](const AttTile<E> &x) {
#pragma unroll
        for (int t = 0; t < NK / 16; t++) {
            const uint32_t key = x.n == NK ? t * 16 + n : min((uint32_t)(t * 16 + n), x.n - 1);
            const uint32_t off = key * kvb + 16 * g;
#pragma unroll
            for (int u = 0; u < S::QR; u++) k[t * S::QR + u] = *(const u32x4e *)((const uint8_t *)x.k + (off + 64 * u));
        }
    };
    auto load_v = [&](const AttTile<E> &x) {
#pragma unroll
        for (int j = 0; j < S::VK; j++) {
            const uint32_t key = x.n == NK ? v_key(j) : min((uint32_t)v_key(j), x.n - 1);
            const uint32_t off = key * kvb + n * (uint32_t)(S::CW * sizeof(E));
#pragma unroll
            for (int h = 0; h < S::VL; h++) {
                if constexpr (!F32 && D == 64) {
                    const u32x2 t = *(const u32x2e *)((const uint8_t *)x.v + off);
                    v[j] = u32x4{t[0], t[1], 0, 0};
                } else {
                    v[j * S::VL + h] = *(const u32x4e *)((const uint8_t *)x.v + (off + h * (uint32_t)(16 * S::CW * sizeof(E))));
                }
            }
        }
    };

    AttTile<E> x = {}, nx = {};
    uint32_t t = w.t0 + wave;
    if (t < w.t1) {
        x = att_tile<E, NK>(w, kv, t);
        load_k(x);
        load_v(x);
    }
    for (; t < w.t1; t += NW) {
        const bool more = t + NW < w.t1;
        if (more) nx = att_tile<E, NK>(w, kv, t + NW);
        f32x4 sc[RB][NK / 16];
#pragma unroll
        for (int b = 0; b < RB; b++)
#pragma unroll
            for (int h = 0; h < NK / 16; h++) {
                sc[b][h] = f32x4{0, 0, 0, 0};
                if constexpr (F32) {  // four chains: shorter sums round less
                    f32x4 part[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        part[c] = f32x4{0, 0, 0, 0};
#pragma unroll
                        for (int u = 0; u < S::QR; u++)
                            part[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[h * S::QR + u][c]), __uint_as_float(q[b][u][c]), part[c], 0, 0, 0);
                    }
                    sc[b][h] = (part[0] + part[1]) + (part[2] + part[3]);
                } else {
#pragma unroll
                    for (int u = 0; u < S::QR; u++) sc[b][h] = AttElem<KIND>::mma16(k[h * S::QR + u], q[b][u], sc[b][h]);
                }
            }
        if (more) load_k(nx);

        u32x4 p16[RB], p16_rest[RB];
        float p32[RB][NK / 4];
#pragma unroll
        for (int b = 0; b < RB; b++) {
            float *p = p32[b];
            float mx = NEG_INF;
#pragma unroll
            for (int h = 0; h < NK / 16; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) p[h * 4 + i] = sc[b][h][i];
            if (x.n < NK || x.ragged) {
                const AttSees sees(w, x, rel[b]);
#pragma unroll
                for (int i = 0; i < NK / 4; i++) p[i] = sees((i / 4) * 16 + 4 * g + i % 4) ? p[i] : NEG_INF;
            }
#pragma unroll
            for (int i = 0; i < NK / 4; i++) mx = fmaxf(mx, p[i]);
            mx = max32(max16(mx)) * a.scale_log2;
            if (__any(mx > mc[b] + RESCALE)) {
                const float to = fmaxf(mx, mc[b]), f = att_shift(mc[b], to);
                mc[b] = to;
                sum[b] *= f;
#pragma unroll
                for (int c = 0; c < S::NA; c++) acc[b][c] *= f;
            }
            const float base = att_base(mc[b]) - LIFT<KIND>;
#pragma unroll
            for (int i = 0; i < NK / 4; i++) {
                p[i] = att_weight<KIND>(p[i], a.scale_log2, base);
                sum[b] += p[i];
            }
            if constexpr (!F32)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t y = AttElem<KIND>::pair(p[2 * i], p[2 * i + 1]);
                    p16[b][i] = y;
                    p16_rest[b][i] = AttElem<KIND>::pair(p[2 * i] - AttElem<KIND>::first(y), p[2 * i + 1] - AttElem<KIND>::second(y));
                }
        }

        // values that no row may see, or only some rows, must not meet a
        // weight of 0 as infinities or NaN, nor any infinity the rest of a
        // weight, whose sign is either
        uint32_t bad = 0;
        bool apart = x.n < NK || x.ragged;
        if constexpr (!F32) {
            typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
            u16x2 top = {0, 0};
#pragma unroll
            for (int i = 0; i < S::VK * S::VL; i++)
#pragma unroll
                for (int e = 0; e < (D == 64 ? 2 : 4); e++)
                    top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, v[i][e] & 0x7FFF7FFFu));
            apart |= __any(!AttElem<KIND>::finite(top[0]) || !AttElem<KIND>::finite(top[1]));
        }
        if (apart) {
#pragma unroll
            for (int j = 0; j < S::VK; j++)
#pragma unroll
                for (int h = 0; h < S::VL; h++) {
                    u32x4 &y = v[j * S::VL + h];
                    if ((uint32_t)v_key(j) >= x.n) y = u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        bool ok;
                        if constexpr (F32) {
                            ok = AttElem<KIND>::finite(y[e]);
                            y[e] = ok ? y[e] : 0;
                        } else {
                            const bool lo = AttElem<KIND>::finite(y[e]), hi = AttElem<KIND>::finite(y[e] >> 16);
                            y[e] &= (lo ? 0xFFFFu : 0u) | (hi ? 0xFFFF0000u : 0u);
                            ok = lo & hi;
                        }
                        bad |= (ok ? 0u : 1u) << v_key(j);
                    }
                }
        }

        if constexpr (F32) {
#pragma unroll
            for (int c = 0; c < S::NA; c++)
#pragma unroll
                for (int b = 0; b < RB; b++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        acc[b][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[j * S::VL + c / 4][c % 4]), p32[b][j], acc[b][c], 0, 0, 0);
        } else {
#pragma unroll
            for (int c = 0; c < S::NA; c++) {
                const int h = c / S::CW, e = c % S::CW / 2;
                u32x4 vt;
#pragma unroll
                for (int j = 0; j < 4; j++)  // keys 2j and 2j + 1 of dimension c
                    vt[j] = __builtin_amdgcn_perm(v[(2 * j + 1) * S::VL + h][e], v[2 * j * S::VL + h][e], c % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int b = 0; b < RB; b++) acc[b][c] = AttElem<KIND>::mma16(vt, p16_rest[b], AttElem<KIND>::mma16(vt, p16[b], acc[b][c]));
            }
        }
        // the keys whose values were taken out, for the rows that see them
        if (apart) {
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) bad |= __shfl_xor(bad, o, 64);
            bad = __builtin_amdgcn_readfirstlane(bad);
            while (bad) {
                const int c = __builtin_ctz(bad);
                bad &= bad - 1;
#pragma unroll
                for (int b = 0; b < RB; b++) {
                    const bool vis = AttSees(w, x, rel[b])(c);
                    float pv = 0.0f;
#pragma unroll
                    for (int i = 0; i < NK / 4; i++) pv = (c / 16) * 4 + c % 4 == i ? p32[b][i] : pv;
                    pv = __shfl(pv, n + 16 * (c % 16 / 4), 64);
#pragma unroll
                    for (int e = 0; e < S::NA; e++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const E y = *(const E *)((const uint8_t *)x.v + (c * kvb + S::dim(e, 4 * g + i) * (uint32_t)sizeof(E)));
                            uint32_t bits;
                            if constexpr (F32) bits = __float_as_uint(y);
                            else bits = y;
                            const float sum_with = acc[b][e][i] + pv * AttElem<KIND>::up(y);
                            acc[b][e][i] = (vis & !AttElem<KIND>::finite(bits)) ? sum_with : acc[b][e][i];
                            __builtin_amdgcn_sched_barrier(0);  // one load at a time: registers for the paths that run
                        }
                }
            }
        }
        if (more) load_v(nx);
        x = nx;
    }

    // The waves' results: their maxima first, then each one's accumulator in
    // units of the common one; the block's threads add up four dimensions at a
    // time. Rows that are not there take no part.
    float (*const l_acc)[ROWS][D + 4] = (float (*)[ROWS][D + 4])lds;
    float2 (*const l_ml)[ROWS] = (float2 (*)[ROWS])(lds + NW * ROWS * (D + 4) * sizeof(float));
#pragma unroll
    for (int b = 0; b < RB; b++) {
        sum[b] = sum32(sum16(sum[b]));
        if (g == 0) l_ml[wave][b * 16 + n] = make_float2(mc[b], sum[b]);
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < RB; b++) {
        if ((uint32_t)(b * 16 + n) >= w.nr) continue;
        float to = NEG_INF;
#pragma unroll
        for (int o = 0; o < NW; o++) to = fmaxf(to, l_ml[o][b * 16 + n].x);
        const float f = att_shift(mc[b], to);
#pragma unroll
        for (int c = 0; c < S::NA; c++) *(f32x4 *)&l_acc[wave][b * 16 + n][c * 16 + 4 * g] = acc[b][c] * f;
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < w.nr * (D / 4); e += NW * 64) {
        const uint32_t row = e / (D / 4), d = e % (D / 4) * 4, rr = w.r0 + row;
        // dimension d: accumulator c and row m of it (S::dim), the next three in c + 1..
        const int m = (int)(d % (16 * S::CW)) / S::CW, c = (int)(d / (16 * S::CW)) * S::CW + (int)d % S::CW;
        float to = NEG_INF, total = 0.0f;
#pragma unroll
        for (int o = 0; o < NW; o++) to = fmaxf(to, l_ml[o][row].x);
#pragma unroll
        for (int o = 0; o < NW; o++) total += l_ml[o][row].y * att_shift(l_ml[o][row].x, to);
        f32x4 y = {0, 0, 0, 0};
#pragma unroll
        for (int o = 0; o < NW; o++)
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] += l_acc[o][row][(c + i) * 16 + m];
        if (w.direct) {
            const float r = w.sees_any(rr) ? 1.0f / total : 0.0f;
            store4<KIND>(a.out, w.at(a, rr, D) + d, y[0] * r, y[1] * r, y[2] * r, y[3] * r);
        } else {
            const size_t slot = w.slot(a, rr);
            if (d == 0) ((float2 *)a.part_ml)[slot] = make_float2(to, total);
            *(f32x4 *)(a.part_acc + slot * D + d) = y;
        }
    }
}

// -------------------------------------------------------------- many rows
// 32 rows per wave, NW waves on the same keys: K and V tiles go through LDS,
// the next tile's loads in flight in registers while this one is multiplied.
// LDS rows are padded so that the operand reads touch every bank once: K's
// 16-byte reads of 32 rows by 16 bytes, 16-bit V's transposing reads (4 keys x
// 32 dimensions per half wave) by 64 bytes.
// 8192 bf16 rows behind a window of 4096, 32 heads over 8 of 128: 450 to 480 us,
// 870 to 930 TFLOP/s (a matrix product of the library's 1218). The matrix cores
// are busy 44 % of it, the vector units, for the exponentials, 46 %; eight waves on
// the same keys took as long, and longer with few rows (64 f32: 46 -> 56 us).
template <int KIND, int D>
struct WideShape {
    static constexpr bool F32 = KIND == AOTK_F32;
    static constexpr int ESZ = F32 ? 4 : 2;
    static constexpr int NK = (F32 || D == 256) ? 32 : 64;
    static constexpr int KS = D + 16 / ESZ;              // LDS row of K, elements
    static constexpr int VS = F32 ? D : D + 32;          // LDS row of V
    static constexpr int QR = F32 ? D / 8 : D / 16;      // 16-byte registers of q
    static constexpr int NA = D / 32;                    // accumulators of 32 dimensions x 32 rows
    static constexpr int CW = F32 ? (D == 64 ? 2 : 4) : 1;
    // dimension of accumulator c, row m of its 32
    static __device__ __forceinline__ int dim(int c, int m) { return F32 ? c / CW * (32 * CW) + m * CW + c % CW : c * 32 + m; }
    static constexpr size_t lds_bytes() { return 2 * (size_t)NK * (KS + VS) * ESZ + 6 * sizeof(uint32_t); }
};

// TWO: 16-bit weights in two parts.
template <int KIND, int D, int NW, bool TWO>
__device__ __forceinline__ void attend_wide(const AttendLaunch &a, bool prefix, uint8_t *lds) {
    typedef WideShape<KIND, D> S;
    typedef typename AttElem<KIND>::elem E;
    constexpr int NK = S::NK, ROWS = 32 * NW, TH = NW * 64;
    constexpr bool F32 = S::F32;
    constexpr int CPR = D * S::ESZ / 16, NCH = NK * CPR / TH;  // 16-byte pieces of a row, per thread
    E *const lk = (E *)lds, *const lv = lk + 2 * NK * S::KS;
    uint32_t (*const l_bad)[2] = (uint32_t (*)[2])(lv + 2 * NK * S::VS);
    const AttJob w = att_job<E, D, ROWS, NK>(a, prefix);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, h = lane >> 5;
    const size_t kv = (size_t)a.n_kv_head * D;
    const uint32_t kvb = a.n_kv_head * (uint32_t)(D * sizeof(E));  // bytes between keys

    const uint32_t rr = w.r0 + min((uint32_t)(wave * 32 + n), w.nr - 1);
    const int rel = w.rel(rr);  // position behind the block's first
    u32x4 q[S::QR];
    {
        const E *src = (const E *)a.q + w.at(a, rr, D);
#pragma unroll
        for (int u = 0; u < S::QR; u++) q[u] = *(const u32x4e *)(src + (F32 ? 8 * u + 4 * h : 16 * u + 8 * h));
    }
    f32x16 acc[S::NA];
#pragma unroll
    for (int c = 0; c < S::NA; c++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[c][i] = 0.0f;
    float mc = NEG_INF, sum = 0.0f;

    u32x4 sk[NCH], sv[NCH];
    // piece e of a thread: row e * TH / CPR behind its first, the same column
    constexpr int RSTEP = TH / CPR;
    static_assert(TH % CPR == 0 && NK % RSTEP == 0, "pieces are whole rows apart");
    const int srow = tid / CPR, scol = tid % CPR * (16 / S::ESZ);
    auto fetch = [&](const AttTile<E> &x) {
        const uint32_t col = scol * (uint32_t)sizeof(E);
        if (x.n == NK) {
            const uint32_t off = srow * kvb + col;
#pragma unroll
            for (int e = 0; e < NCH; e++) {
                sk[e] = *(const u32x4e *)((const uint8_t *)x.k + (off + e * RSTEP * kvb));
                sv[e] = *(const u32x4e *)((const uint8_t *)x.v + (off + e * RSTEP * kvb));
            }
        } else {  // keys past the end: the last one
#pragma unroll
            for (int e = 0; e < NCH; e++) {
                const uint32_t off = min((uint32_t)(srow + e * RSTEP), x.n - 1) * kvb + col;
                sk[e] = *(const u32x4e *)((const uint8_t *)x.k + off);
                sv[e] = *(const u32x4e *)((const uint8_t *)x.v + off);
            }
        }
    };
    // into the buffer; values past the tile's end become 0, and in a tile
    // that rows see differently, or whose weights have two parts, those not
    // finite do, their keys noted
    auto put = [&](const AttTile<E> &x, int buf, int slot) {
        bool apart = x.ragged;
        if constexpr (TWO) {
            typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
            u16x2 top = {0, 0};
#pragma unroll
            for (int e = 0; e < NCH; e++)
#pragma unroll
                for (int c = 0; c < 4; c++) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, sv[e][c] & 0x7FFF7FFFu));
            apart |= __any(!AttElem<KIND>::finite(top[0]) || !AttElem<KIND>::finite(top[1]));
        }
#pragma unroll
        for (int e = 0; e < NCH; e++) {
            const int row = srow + e * RSTEP;
            if (x.n < NK || apart) {
                u32x4 &y = sv[e];
                bool bad = false;
                if ((uint32_t)row >= x.n) y = u32x4{0, 0, 0, 0};
                else if (apart)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        if constexpr (F32) {
                            const bool ok = AttElem<KIND>::finite(y[c]);
                            y[c] = ok ? y[c] : 0;
                            bad |= !ok;
                        } else {
                            const bool lo = AttElem<KIND>::finite(y[c]), hi = AttElem<KIND>::finite(y[c] >> 16);
                            y[c] &= (lo ? 0xFFFFu : 0u) | (hi ? 0xFFFF0000u : 0u);
                            bad |= !lo || !hi;
                        }
                    }
                if (bad) atomicOr(&l_bad[slot][row >> 5], 1u << (row & 31));
            }
            *(u32x4 *)(lk + (buf * NK + row) * S::KS + scol) = sk[e];
            *(u32x4 *)(lv + (buf * NK + row) * S::VS + scol) = sv[e];
        }
    };

    // V's operands of step vi: f32, one key per half (accumulator register vi's)
    // and four dimensions a lane and load; 16 bits, 16 keys. There lane l of a
    // transposing read addresses key l % 16 / 4, dimensions 4 (l % 4).. of its 16
    // lanes' 4 x 16 piece, and receives dimension l % 16 of the 4 keys.
    constexpr int VN = F32 ? 16 : NK / 16, VG = F32 ? (S::NA + 3) / 4 : S::NA;
    auto read_v = [&](int buf, int vi, u32x4 *f) {
        if constexpr (F32) {
            const float *row = (const float *)lv + (buf * NK + 8 * (vi / 4) + 4 * h + vi % 4) * S::VS + n * S::CW;
#pragma unroll
            for (int c = 0; c < VG; c++) {
                if constexpr (S::CW == 2) {
                    const u32x2 y = *(const u32x2 *)row;
                    f[c] = u32x4{y[0], y[1], 0, 0};
                } else {
                    f[c] = *(const u32x4 *)(row + c * 128);
                }
            }
        } else {
            typedef __attribute__((address_space(3))) i16x4 *lds_i16x4;
            const E *at = lv + (buf * NK + vi * 16 + 4 * h + (lane >> 2 & 3)) * S::VS + (lane >> 4 & 1) * 16 + (lane & 3) * 4;
#pragma unroll
            for (int c = 0; c < VG; c++) {
                const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(at + c * 32)));
                const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(at + c * 32 + 8 * S::VS)));
                f[c] = u32x4{lo[0], lo[1], hi[0], hi[1]};
            }
        }
    };

    if (tid < 6) l_bad[tid >> 1][tid & 1] = 0;
    AttTile<E> x = {}, nx = {};
    __syncthreads();
    if (w.t0 < w.t1) {
        x = att_tile<E, NK>(w, kv, w.t0);
        fetch(x);
        put(x, 0, 0);
    }
    __syncthreads();
    int slot = 0;
    for (uint32_t t = w.t0; t < w.t1; t++) {
        const int buf = (t - w.t0) & 1;
        const bool more = t + 1 < w.t1;
        if (more) {
            nx = att_tile<E, NK>(w, kv, t + 1);
            fetch(nx);
        }
        // Operands come from LDS a group ahead of the products that take them.
        // (Pinning that order, and weaving the weights' vector instructions into
        // the products of the other half of the tile, measured no faster: two
        // waves a SIMD take turns by themselves.)
        constexpr int P = NK / 32, KG = S::QR / 4;
        f32x16 sc[P];
        uint32_t p16[P * 8], p16_rest[P * 8];  // 16 bits: the weights, two a word, in sc's order
        u32x4 kf[2][4], vf[2][VG];
        const E *const krow = lk + (buf * NK + n) * S::KS + (F32 ? 4 * h : 8 * h);
        auto read_k = [&](int kb, int gi) {
#pragma unroll
            for (int e = 0; e < 4; e++) kf[(kb * KG + gi) & 1][e] = *(const u32x4 *)(krow + kb * 32 * S::KS + (gi * 4 + e) * (F32 ? 8 : 16));
        };
        auto scores = [&](int kb, int gi) {
            if (gi == 0)
#pragma unroll
                for (int i = 0; i < 16; i++) sc[kb][i] = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const u32x4 kk = kf[(kb * KG + gi) & 1][e], qq = q[gi * 4 + e];
                if constexpr (F32) {
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        sc[kb] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kk[c]), __uint_as_float(qq[c]), sc[kb], 0, 0, 0);
                } else {
                    sc[kb] = AttElem<KIND>::mma32(kk, qq, sc[kb]);
                }
            }
        };
        auto rescale = [&]() {
            if (x.n < NK || x.ragged) {
                const AttSees sees(w, x, rel);
#pragma unroll
                for (int kb = 0; kb < P; kb++)
#pragma unroll
                    for (int i = 0; i < 16; i++) sc[kb][i] = sees(kb * 32 + 8 * (i / 4) + 4 * h + i % 4) ? sc[kb][i] : NEG_INF;
            }
            float mx = NEG_INF;
#pragma unroll
            for (int kb = 0; kb < P; kb++)
#pragma unroll
                for (int i = 0; i < 16; i++) mx = fmaxf(mx, sc[kb][i]);
            mx = max32(mx) * a.scale_log2;
            if (__any(mx > mc + RESCALE)) {
                const float to = fmaxf(mx, mc), f = att_shift(mc, to);
                mc = to;
                sum *= f;
#pragma unroll
                for (int c = 0; c < S::NA; c++)
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[c][i] *= f;
            }
        };
        auto weights = [&]() {
            const float base = att_base(mc) - LIFT<KIND>;
#pragma unroll
            for (int kb = 0; kb < P; kb++)
#pragma unroll
                for (int i = 0; i < 16; i++) sc[kb][i] = att_weight<KIND>(sc[kb][i], a.scale_log2, base);
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // short chains of sums
#pragma unroll
            for (int i = 0; i < P * 8; i++) {
                const float x = sc[i / 8][i % 8 * 2], y = sc[i / 8][i % 8 * 2 + 1];
                if constexpr (F32) {
                    part[i % 4] += x + y;
                } else {
                    p16[i] = AttElem<KIND>::pair(x, y);
                    if constexpr (TWO) {
                        p16_rest[i] = AttElem<KIND>::pair(x - AttElem<KIND>::first(p16[i]), y - AttElem<KIND>::second(p16[i]));
                        part[i % 4] += x + y;
                    } else {
                        part[i % 4] = AttElem<KIND>::add_pair(p16[i], part[i % 4]);
                    }
                }
            }
            sum += (part[0] + part[1]) + (part[2] + part[3]);
        };
        auto values = [&](int vi) {
            if constexpr (F32) {
#pragma unroll
                for (int c = 0; c < S::NA; c++)
                    acc[c] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(vf[vi & 1][c / 4][c % 4]), sc[0][vi], acc[c], 0, 0, 0);
            } else {
                const u32x4 p = {p16[vi * 4], p16[vi * 4 + 1], p16[vi * 4 + 2], p16[vi * 4 + 3]};
#pragma unroll
                for (int c = 0; c < S::NA; c++) acc[c] = AttElem<KIND>::mma32(vf[vi & 1][c], p, acc[c]);
                if constexpr (TWO) {
                    const u32x4 r = {p16_rest[vi * 4], p16_rest[vi * 4 + 1], p16_rest[vi * 4 + 2], p16_rest[vi * 4 + 3]};
#pragma unroll
                    for (int c = 0; c < S::NA; c++) acc[c] = AttElem<KIND>::mma32(vf[vi & 1][c], r, acc[c]);
                }
            }
        };
        read_k(0, 0);
#pragma unroll
        for (int ki = 0; ki < P * KG; ki++) {
            if (ki + 1 < P * KG) read_k((ki + 1) / KG, (ki + 1) % KG);
            scores(ki / KG, ki % KG);
        }
        read_v(buf, 0, vf[0]);
        rescale();
        weights();
#pragma unroll
        for (int vi = 0; vi < VN; vi++) {
            if (vi + 1 < VN) read_v(buf, vi + 1, vf[(vi + 1) & 1]);
            values(vi);
        }
        if (x.ragged || TWO) {
            for (int half = 0; half < NK / 32; half++) {
                uint32_t bad = __builtin_amdgcn_readfirstlane(l_bad[slot][half]);
                const AttSees sees(w, x, rel);
                while (bad) {
                    const int c = __builtin_ctz(bad) + 32 * half;
                    bad &= bad - 1;
                    float pv = 0.0f;  // the key's weight
#pragma unroll
                    for (int i = 0; i < P * 16; i++) {
                        float y;
                        if constexpr (F32 || TWO) y = sc[i / 16][i % 16];
                        else y = i % 2 ? AttElem<KIND>::second(p16[i / 2]) : AttElem<KIND>::first(p16[i / 2]);
                        pv = i == (c / 32) * 16 + c % 32 / 8 * 4 + c % 4 ? y : pv;
                    }
                    pv = __shfl(pv, n + 32 * (c / 4 % 2), 64);
                    const bool vis = sees(c);
#pragma unroll
                    for (int e = 0; e < S::NA; e++)
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const E y = *(const E *)((const uint8_t *)x.v + (c * kvb + S::dim(e, 8 * (i / 4) + 4 * h + i % 4) * (uint32_t)sizeof(E)));
                            uint32_t bits;
                            if constexpr (F32) bits = __float_as_uint(y);
                            else bits = y;
                            const float sum_with = acc[e][i] + pv * AttElem<KIND>::up(y);
                            acc[e][i] = (vis & !AttElem<KIND>::finite(bits)) ? sum_with : acc[e][i];
                            __builtin_amdgcn_sched_barrier(0);
                        }
                }
            }
        }
        // the slot after next is free: it was read in the last round, and is
        // written again after this round's barrier
        const int next = slot == 2 ? 0 : slot + 1, after = next == 2 ? 0 : next + 1;
        if (tid < 2) l_bad[after][tid] = 0;
        if (more) put(nx, buf ^ 1, next);
        x = nx;
        slot = next;
        __syncthreads();
    }
    sum = sum32(sum);
    if ((uint32_t)(wave * 32 + n) >= w.nr) return;
    auto four = [&](auto f) {  // f(dimension, four accumulated values from it on)
#pragma unroll
        for (int c = 0; c < S::NA; c += F32 ? S::CW : 1)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int m = 8 * (i / 4) + 4 * h;
                if constexpr (!F32) f(S::dim(c, m), acc[c][i], acc[c][i + 1], acc[c][i + 2], acc[c][i + 3]);
                else if constexpr (S::CW == 4)
#pragma unroll
                    for (int e = 0; e < 4; e++) f(S::dim(c, m + e), acc[c][i + e], acc[c + 1][i + e], acc[c + 2][i + e], acc[c + 3][i + e]);
                else
#pragma unroll
                    for (int e = 0; e < 4; e += 2) f(S::dim(c, m + e), acc[c][i + e], acc[c + 1][i + e], acc[c][i + e + 1], acc[c + 1][i + e + 1]);
            }
    };
    if (w.direct) {
        const float r = w.sees_any(rr) ? 1.0f / sum : 0.0f;
        const size_t at = w.at(a, rr, D);
        four([&](int d, float e0, float e1, float e2, float e3) { store4<KIND>(a.out, at + d, e0 * r, e1 * r, e2 * r, e3 * r); });
    } else {
        const size_t slot_at = w.slot(a, rr);
        if (h == 0) ((float2 *)a.part_ml)[slot_at] = make_float2(mc, sum);
        four([&](int d, float e0, float e1, float e2, float e3) { *(f32x4 *)(a.part_acc + slot_at * D + d) = f32x4{e0, e1, e2, e3}; });
    }
}

// ---------------------------------------------------------------- kernels
// The prefix's blocks come first, over the rows of all sequences, then those of
// the sequences' own ranges. Both in one launch: the prefix's many rows wait
// for the matrix cores, the tails' few rows for memory, and neither alone fills
// the chip. P and O: 16-row tiles of attend_narrow (1, 2) or 32-row waves of
// attend_wide (3: two waves, 4: four).
template <int KIND, int D, int SHAPE, int NW, bool TWO>
__device__ __forceinline__ void attend_shape(const AttendLaunch &a, bool prefix, uint8_t *lds) {
    if constexpr (SHAPE <= 2) attend_narrow<KIND, D, NW, SHAPE>(a, prefix, lds);
    else attend_wide<KIND, D, NW, TWO>(a, prefix, lds);
}

constexpr int att_waves(int p) { return p == 3 ? 2 : 4; }

template <int KIND, int D, int SHAPE, int NW>
constexpr size_t att_lds() {
    if constexpr (SHAPE <= 2) return NarrowShape<KIND, D>::template lds_bytes<NW, SHAPE>();
    else return WideShape<KIND, D>::lds_bytes();
}

template <int KIND, int D, int P, int O>
__global__ __launch_bounds__(64 * att_waves(P), D == 256 || P == 3 ? 1 : 2) void k_attend(AttendLaunch a) {
    extern __shared__ __align__(16) uint8_t lds[];
    const bool prefix = blockIdx.x < a.prefix_blocks;
    if constexpr (P == O) {
        attend_shape<KIND, D, P, att_waves(P), false>(a, prefix, lds);
    } else {
        if (prefix) attend_shape<KIND, D, P, att_waves(P), KIND != AOTK_F32>(a, true, lds);
        else attend_shape<KIND, D, O, att_waves(P), false>(a, false, lds);
    }
}

// ------------------------------------------------------------------- join
// WAVES waves per row and query head: the runs of the prefix, then those of the
// sequence's own range. A lane holds the weight of every 64th run; each wave
// sums every WAVES-th run's accumulators, four loads in flight. Bound by its chain
// of loads: 57 runs of 32 rows 8.2 us by one wave a row, 4.4 by sixteen; 2048 rows
// of 12 runs, 13 MB, 5.7 us. (In the last block of a kv head instead of a launch:
// 25 -> 33 us for a call of 4 sequences behind 512.)
template <int KIND, int D, int WAVES>
__global__ __launch_bounds__(WAVES > 4 ? 64 * WAVES : 256) void k_join(AttendLaunch a, uint32_t prefix_chunks, uint32_t total, uint32_t row_begin) {
    constexpr int N = D / 64;
    typedef float vec __attribute__((ext_vector_type(N)));
    constexpr int ROWS = WAVES > 4 ? 1 : 4 / WAVES;  // of a block
    __shared__ float l_acc[ROWS * WAVES][D];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % WAVES;
    const uint32_t item = blockIdx.x * ROWS + wave / WAVES;
    const uint32_t row = row_begin + item / a.n_head, head = item % a.n_head;
    const bool le = lane < (int)a.n_seq && a.seq[lane].row0 <= row;
    const uint32_t si = (uint32_t)__builtin_amdgcn_readfirstlane(__popcll(__ballot(le)) - 1);
    const AttendPlace s = a.seq[si];
    const uint32_t i = row - s.row0;
    const bool mine = i < s.rows && (s.chunks > 1 || a.joined);
    const uint32_t n = mine ? prefix_chunks + s.chunks : 0;
    auto slot = [&](uint32_t c) {
        return (c < prefix_chunks ? (size_t)c * total + row : s.part0 + (size_t)(c - prefix_chunks) * s.rows + i) * a.n_head + head;
    };
    const float2 *ml = (const float2 *)a.part_ml;
    float mx = NEG_INF;
    for (uint32_t c = lane; c < n; c += 64) mx = fmaxf(mx, ml[slot(c)].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, shfl_xor(mx, o));
    vec acc = 0.0f;
    float sum = 0.0f;
    for (uint32_t c0 = 0; c0 < n; c0 += 64) {
        float w = 0.0f;
        if (c0 + lane < n) {
            const float2 x = ml[slot(c0 + lane)];
            w = att_shift(x.x, mx);
            sum += x.y * w;
        }
        const uint32_t nc = min(n - c0, 64u);
        for (uint32_t c = part; c < nc; c += 4 * WAVES) {
            vec y[4];
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t ce = min(c + e * WAVES, nc - 1);
                y[e] = *(const vec *)(a.part_acc + slot(c0 + ce) * D + lane * N);
                f[e] = c + e * WAVES < nc ? readlane_f(w, ce) : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (c + e * WAVES < nc) acc += y[e] * f[e];
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += shfl_xor(sum, o);
    if constexpr (WAVES > 1) {
        *(vec *)&l_acc[wave][lane * N] = acc;
        __syncthreads();
        if (part != 0) return;
#pragma unroll
        for (int e = 1; e < WAVES; e++) acc += *(const vec *)&l_acc[wave + e][lane * N];
    }
    if (!mine) return;
    const int64_t p = (int64_t)s.len - s.rows + i;
    const float r = prefix_chunks > 0 || a.range[0].na > 0 || p >= 0 ? 1.0f / sum : 0.0f;
    const size_t at = ((size_t)row * a.n_head + head) * D + lane * N;
#pragma unroll
    for (int e = 0; e < N; e++) {
        if constexpr (KIND == AOTK_F32) ((float *)a.out)[at + e] = acc[e] * r;
        else ((uint16_t *)a.out)[at + e] = (uint16_t)AttElem<KIND>::pair(acc[e] * r, 0.0f);
    }
}

// ----------------------------------------------------------------- launch
template <int KIND, int D, int P, int O>
static void att_start(const AttendLaunch &a, uint32_t blocks, hipStream_t s) {
    constexpr size_t lp = att_lds<KIND, D, P, att_waves(P)>(), lo = att_lds<KIND, D, O, att_waves(P)>(), lds = lp > lo ? lp : lo;
    static const hipError_t more = hipFuncSetAttribute((const void *)k_attend<KIND, D, P, O>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    (void)more;  // a launch that it keeps from starting reports the error
    k_attend<KIND, D, P, O><<<blocks, 64 * att_waves(P), lds, s>>>(a);
}

template <int KIND, int D>
static void att_launch_d(int p, int o, const AttendLaunch &a, uint32_t blocks, hipStream_t s) {
    switch (p * 8 + o) {
    case 1 * 8 + 1: return att_start<KIND, D, 1, 1>(a, blocks, s);
    case 2 * 8 + 2:
        if constexpr (D < 256) return att_start<KIND, D, 2, 2>(a, blocks, s);
        break;
    case 3 * 8 + 1: return att_start<KIND, D, 3, 1>(a, blocks, s);
    case 3 * 8 + 2:
        if constexpr (KIND != AOTK_F32 && D < 256) return att_start<KIND, D, 3, 2>(a, blocks, s);
        break;
    case 3 * 8 + 3: return att_start<KIND, D, 3, 3>(a, blocks, s);
    case 4 * 8 + 1: return att_start<KIND, D, 4, 1>(a, blocks, s);
    case 4 * 8 + 2:
        if constexpr (D < 256) return att_start<KIND, D, 4, 2>(a, blocks, s);
        break;
    case 4 * 8 + 4: return att_start<KIND, D, 4, 4>(a, blocks, s);
    }
}

template <int KIND>
void att_launch_kind(int head_dim, int p, int o, const AttendLaunch &a, uint32_t blocks, hipStream_t s) {
    if (head_dim == 64) att_launch_d<KIND, 64>(p, o, a, blocks, s);
    else if (head_dim == 128) att_launch_d<KIND, 128>(p, o, a, blocks, s);
    else att_launch_d<KIND, 256>(p, o, a, blocks, s);
}

template <int KIND>
void att_join_kind(int head_dim, const AttendLaunch &a, uint32_t prefix_chunks, uint32_t total, uint32_t first_row, uint64_t items, uint32_t runs, hipStream_t s) {
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (runs >= 32) k_join<KIND, D, 16><<<(unsigned)items, 1024, 0, s>>>(a, prefix_chunks, total, first_row);
        else if (runs >= 8) k_join<KIND, D, 4><<<(unsigned)items, 256, 0, s>>>(a, prefix_chunks, total, first_row);
        else k_join<KIND, D, 1><<<(unsigned)((items + 3) / 4), 256, 0, s>>>(a, prefix_chunks, total, first_row);
    };
    if (head_dim == 64) go(std::integral_constant<int, 64>());
    else if (head_dim == 128) go(std::integral_constant<int, 128>());
    else go(std::integral_constant<int, 256>());
}

}  // namespace aotk
