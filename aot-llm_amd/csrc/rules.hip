// rules.hip - rules on logits before a token is picked: penalties for the
// tokens of a history, sparse biases, a mask of allowed tokens, and the
// greedy pick of what is left, for a batch of rows in one pass.
//
// For token t of a row, c = occurrences of t in the row's history:
//   y = x
//   c > 0:  y = (x > 0 ? x / repetition : x * repetition) - (presence + frequency * c)
//   biased: y = y + bias of the last entry that names t
//   t not allowed: y = -inf
// in f32, each operation rounded once (the build never contracts), and rounded
// to the logits' type at the end. Rows differ in every rule, so each row's
// rules travel in the launch's arguments.
//
// One read and one write of the logits bound it: 256 x 262144 bf16, 268 MB, 67 us
// (4.1 TB/s; a large copy reaches 6.2), 64 x 128256 f32 18 us, 1 x 32000 6.0 us.
//
// A block takes slices of RULE_SLICE tokens of one row. What names tokens
// in list order (history, biases) is turned into per-token tables in LDS:
// every block scans the row's whole lists and keeps the entries of its slice,
// counting with integer adds and taking the last bias by an integer maximum,
// so no result depends on the order in which threads arrive.
#include "device.hpp"
#include "internal.hpp"

namespace aotk {

constexpr int RULE_THREADS = 512;
constexpr int RULE_PER = RULE_SLICE / RULE_THREADS;  // values per thread

typedef uint32_t u32x4a4 __attribute__((ext_vector_type(4), aligned(4)));

// A thread's piece: 16 bytes of a row, at any multiple of the element size
// (rows start anywhere), as four words.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4a2 __attribute__((ext_vector_type(4), aligned(2)));

template <int KIND>
struct RuleKind {
    typedef uint16_t elem;
    static constexpr int N = 8;  // values of a piece
    static constexpr uint32_t NONE = KIND == AOTK_F16 ? 0xFC00u : 0xFF80u;  // -inf
    static __device__ __forceinline__ float up(uint32_t x) { return KIND == AOTK_F16 ? f16_to_f32(x) : bf16_to_f32(x & 0xFFFFu); }
    // one conversion, to nearest even (overflow to infinity)
    static __device__ __forceinline__ uint32_t down(float x) {
        if constexpr (KIND == AOTK_F16) return __builtin_bit_cast(uint16_t, (_Float16)x);
        else return f32_to_bf16(x);
    }
    static __device__ __forceinline__ float get(const u32x4 &x, int i) { return up(i & 1 ? x[i / 2] >> 16 : x[i / 2]); }
    static __device__ __forceinline__ void set(u32x4 &x, int i, float v) {
        x[i / 2] = i & 1 ? (x[i / 2] & 0xFFFFu) | (down(v) << 16) : (x[i / 2] & 0xFFFF0000u) | down(v);
    }
    // values whose bit is 0 become -inf: bits to fields of ones, two a word
    static __device__ __forceinline__ void allow(u32x4 &x, uint32_t bits) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t lo = (uint32_t)((int)(bits << (31 - 2 * i)) >> 31), hi = (uint32_t)((int)(bits << (30 - 2 * i)) >> 31);
            const uint32_t m = (lo & 0xFFFFu) | (hi & 0xFFFF0000u);
            x[i] = (x[i] & m) | ((NONE << 16 | NONE) & ~m);
        }
    }
};
template <>
struct RuleKind<AOTK_F32> {
    typedef float elem;
    static constexpr int N = 4;
    static __device__ __forceinline__ float get(const u32x4 &x, int i) { return __uint_as_float(x[i]); }
    static __device__ __forceinline__ void set(u32x4 &x, int i, float v) { x[i] = __float_as_uint(v); }
    static __device__ __forceinline__ void allow(u32x4 &x, uint32_t bits) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = (bits >> i) & 1u ? x[i] : 0xFF800000u;
    }
};

// Pick key: the value's order in the high word, the complement of the token
// in the low one (the maximum is the largest value's lowest token). 0 stands
// for no token: NaN and -inf are never picked. Zeros of both signs are equal.
__device__ __forceinline__ uint64_t rule_key(float y, uint32_t t) {
    const uint32_t b = __float_as_uint(y + 0.0f);
    const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((uint64_t)o << 32) | (uint32_t)~t;
}

__device__ __forceinline__ uint64_t wave_max_key(uint64_t k) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor((unsigned long long)k, o, 64);
        k = other > k ? other : k;
    }
    return k;
}

// A thread's four entries of a list of n from place i on.
__device__ __forceinline__ u32x4a4 rule_four(const uint32_t *list, uint32_t n, uint32_t i) {
    u32x4a4 x = {0, 0, 0, 0};
    if (i < n && n - i >= 4) x = *(const u32x4a4 *)(list + i);
    else
#pragma unroll
        for (uint32_t e = 0; e < 4; e++)
            if (i + e < n) x[e] = list[i + e];
    return x;
}

// f(token of the slice, place in the list) for the entries that name the
// block's slice. `first` holds the thread's first four. (Four loads in flight
// instead of one: the registers cost two of four resident blocks, 64 x 128256
// f32 18 -> 23 us.)
template <typename F>
__device__ __forceinline__ void rule_list(const uint32_t *list, uint32_t n, uint32_t base, u32x4a4 first, F f) {
    for (uint32_t i = threadIdx.x * 4; i < n; i += RULE_THREADS * 4) {
        if (i >= RULE_THREADS * 4) first = rule_four(list, n, i);
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
            const uint32_t t = first[e] - base;
            if (i + e < n && t < (uint32_t)RULE_SLICE) f(t, i + e);
        }
    }
}

// A block takes every gridDim.x-th slice of its row, the next slice's logits and
// mask words in flight while one is worked on; the heads of the lists stay in
// registers. The lists' tokens of the slice get a bit each, so that a thread
// asks once for its whole piece whether any rule names a value of it: nearly
// always none does, and the piece is masked and stored as loaded. `tables`: what
// the launch's rows need, 1 a count per token, 2 a bias per token (16 KB of LDS
// each).
//
// The pick: every block raises its row's key by an atomic maximum and counts
// itself in; the last one takes the key and leaves key and count at 0 for the
// next call. Both words change by atomics only, which meet behind the XCDs'
// caches, and a block counts itself after its key has returned from there: no
// cache is flushed for it. (A launch of its own for the picks: 3.5 us more.)
template <int KIND, typename ROWS>
__global__ __launch_bounds__(RULE_THREADS) void k_rules(RuleArgs a, ROWS rows) {
    typedef RuleKind<KIND> K;
    typedef typename K::elem elem;
    constexpr int N = K::N, G = RULE_PER / N;
    extern __shared__ __align__(16) uint32_t tables[];
    __shared__ uint32_t named[RULE_SLICE / 32];
    __shared__ uint64_t best[RULE_THREADS / 64];
    const aotk_logits_rule r = rows.rule[blockIdx.y];
    const size_t row = blockIdx.y;
    const int tid = threadIdx.x;
    const elem *src = (const elem *)a.logits + row * a.stride;
    elem *dst = (elem *)a.out + row * a.stride;
    uint32_t *const cnt = tables, *const last = tables + (a.tables & 1 ? RULE_SLICE : 0);
    const bool pen = r.hist_len > 0 && (r.repetition != 1.0f || r.presence != 0.0f || r.frequency != 0.0f);
    const bool biased = r.bias_len > 0;
    const uint32_t *mask = r.mask >= 0 ? a.mask + (size_t)r.mask * ((a.vocab + 31) / 32) : nullptr;

    auto fetch = [&](uint32_t base, u32x4 *x, uint32_t *word) {
#pragma unroll
        for (int g = 0; g < G; g++) {
            const uint32_t t = base + (g * RULE_THREADS + tid) * N;
            x[g] = u32x4{0, 0, 0, 0};
            word[g] = ~0u;
            if (t >= a.vocab) continue;
            if (t + N <= a.vocab) {
                x[g] = *(const u32x4a2 *)(src + t);
            } else {  // the row ends inside the piece
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (t + i < a.vocab) {
                        if constexpr (N == 4) x[g][i] = __float_as_uint(src[t + i]);
                        else x[g][i / 2] |= (uint32_t)src[t + i] << (i % 2 * 16);
                    }
            }
            if (mask) word[g] = mask[t / 32] >> (t % 32);
        }
    };
    const uint32_t slices = (a.vocab + RULE_SLICE - 1) / RULE_SLICE;
    u32x4 x[G], nx[G];
    uint32_t word[G], nword[G];
    fetch(blockIdx.x * (uint32_t)RULE_SLICE, x, word);
    const u32x4a4 h0 = pen ? rule_four(a.hist + r.hist_off, r.hist_len, tid * 4) : u32x4a4{0, 0, 0, 0};
    const u32x4a4 b0 = biased ? rule_four(a.bias_id + r.bias_off, r.bias_len, tid * 4) : u32x4a4{0, 0, 0, 0};
    float top = -__builtin_inff();
    uint32_t top_at = 0;
    for (uint32_t slice = blockIdx.x; slice < slices; slice += gridDim.x) {
        const uint32_t base = slice * (uint32_t)RULE_SLICE;
        if (pen || biased) {
            const u32x4 zero = {0, 0, 0, 0};
            for (int i = tid * 4; i < RULE_SLICE; i += RULE_THREADS * 4) {
                if (pen) *(u32x4 *)(cnt + i) = zero;
                if (biased) *(u32x4 *)(last + i) = zero;
            }
            if (tid < RULE_SLICE / 32) named[tid] = 0;
            __syncthreads();
        }
        if (slice + gridDim.x < slices) fetch((slice + gridDim.x) * (uint32_t)RULE_SLICE, nx, nword);
        if (pen || biased) {
            if (pen)
                rule_list(a.hist + r.hist_off, r.hist_len, base, h0, [&](uint32_t t, uint32_t) {
                    atomicAdd(&cnt[t], 1u);
                    atomicOr(&named[t / 32], 1u << (t % 32));
                });
            if (biased)
                rule_list(a.bias_id + r.bias_off, r.bias_len, base, b0, [&](uint32_t t, uint32_t i) {
                    atomicMax(&last[t], i + 1);
                    atomicOr(&named[t / 32], 1u << (t % 32));
                });
            __syncthreads();
        }
#pragma unroll
        for (int g = 0; g < G; g++) {
            const uint32_t ts = (g * RULE_THREADS + tid) * N, t = base + ts;
            if (t >= a.vocab) continue;
            const uint32_t left = a.vocab - t;
            if (pen || biased) {
                const uint32_t who = (named[ts / 32] >> (ts % 32)) & ((1u << N) - 1);
                if (who)
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        if (!((who >> i) & 1u)) continue;
                        float v = K::get(x[g], i);
                        const uint32_t c = pen ? cnt[ts + i] : 0, e = biased ? last[ts + i] : 0;
                        if (c) v = (v > 0.0f ? v / r.repetition : v * r.repetition) - (r.presence + r.frequency * (float)c);
                        if (e) v = v + a.bias[(size_t)r.bias_off + e - 1];
                        K::set(x[g], i, v);
                    }
            }
            uint32_t bits = word[g];
            if (left < N) bits &= (1u << left) - 1;  // nothing behind the row's end is picked
            if (mask || left < N) K::allow(x[g], bits);
            if (left >= N) {
                *(u32x4a2 *)(dst + t) = x[g];
            } else {
#pragma unroll
                for (int i = 0; i < N; i++)
                    if ((uint32_t)i < left) {
                        if constexpr (N == 4) dst[t + i] = __uint_as_float(x[g][i]);
                        else dst[t + i] = (uint16_t)(x[g][i / 2] >> (i % 2 * 16));
                    }
            }
            if (a.tokens) {  // NaN is passed over; the lowest of equal values stays
                float m = -__builtin_inff();
#pragma unroll
                for (int i = 0; i < N; i++) m = fmaxf(m, K::get(x[g], i));
                if (m > top) {
                    top = m;
#pragma unroll
                    for (int i = N - 1; i >= 0; i--) top_at = K::get(x[g], i) == m ? t + i : top_at;
                }
            }
        }
#pragma unroll
        for (int g = 0; g < G; g++) {
            x[g] = nx[g];
            word[g] = nword[g];
        }
        if (pen || biased) __syncthreads();  // the tables are read before the next slice's
    }
    if (!a.tokens) return;
    uint64_t key = wave_max_key(top > -__builtin_inff() ? rule_key(top, top_at) : 0);
    if ((tid & 63) == 0) best[tid >> 6] = key;
    __syncthreads();
    if (tid != 0) return;
    for (int w = 1; w < RULE_THREADS / 64; w++) key = best[w] > key ? best[w] : key;
    if (gridDim.x > 1) {
        RulePick *p = a.picks + row;
        const uint64_t before = __hip_atomic_fetch_max(&p->key, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" : : "v"((uint32_t)before) : "memory");
        if (__hip_atomic_fetch_add(&p->done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != gridDim.x - 1) return;
        key = __hip_atomic_exchange(&p->key, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&p->done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    a.tokens[row] = key ? ~(uint32_t)key : 0xFFFFFFFFu;
}

// Blocks of a row: four a CU over all rows, every one the same number of slices.
static unsigned rules_blocks(size_t rows, size_t vocab) {
    const size_t slices = (vocab + RULE_SLICE - 1) / RULE_SLICE;
    const size_t want = (1024 + rows - 1) / rows, each = slices > want ? (slices + want - 1) / want : 1;
    return (unsigned)((slices + each - 1) / each);
}

// Few rows' rules travel in the launch's arguments, more are read where the
// caller keeps them (1 x 32000 f32: 4.7 against 6.0 us in host memory; 256 rows
// in the arguments of three launches: 92 against 65 us).
struct RuleFew {
    aotk_logits_rule rule[RULE_FEW];
};
struct RuleMany {
    const aotk_logits_rule *rule;
};

template <typename ROWS>
static void rules_start(int kind, const RuleArgs &a, const ROWS &rows, unsigned blocks, unsigned n, hipStream_t s) {
    const size_t lds = ((a.tables & 1) + (a.tables >> 1)) * RULE_SLICE * sizeof(uint32_t);
    const dim3 grid(blocks, n);
    switch (kind) {
    case AOTK_F32: k_rules<AOTK_F32><<<grid, RULE_THREADS, lds, s>>>(a, rows); break;
    case AOTK_F16: k_rules<AOTK_F16><<<grid, RULE_THREADS, lds, s>>>(a, rows); break;
    default: k_rules<AOTK_BF16><<<grid, RULE_THREADS, lds, s>>>(a, rows); break;
    }
}

void launch_rules(int kind, RuleArgs a, const aotk_logits_rule *rules, size_t rows, hipStream_t s) {
    const unsigned blocks = rules_blocks(rows, a.vocab);
    a.tables = 0;
    for (size_t i = 0; i < rows; i++) a.tables |= (rules[i].hist_len ? 1u : 0u) | (rules[i].bias_len ? 2u : 0u);
    if (rows <= (size_t)RULE_FEW) {
        RuleFew few = {};
        for (size_t i = 0; i < rows; i++) few.rule[i] = rules[i];
        return rules_start(kind, a, few, blocks, (unsigned)rows, s);
    }
    for (size_t r0 = 0; r0 < rows; r0 += 65535) {
        RuleArgs p = a;
        p.logits = (const uint8_t *)a.logits + r0 * a.stride * type_size(kind);
        p.out = (uint8_t *)a.out + r0 * a.stride * type_size(kind);
        p.tokens = a.tokens ? a.tokens + r0 : nullptr;
        p.picks = a.picks ? a.picks + r0 : nullptr;
        rules_start(kind, p, RuleMany{a.rules + r0}, blocks, (unsigned)(rows - r0 < 65535 ? rows - r0 : 65535), s);
    }
}

}  // namespace aotk
