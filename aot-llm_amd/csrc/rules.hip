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
// A block takes one slice of RULE_SLICE tokens of one row. What names tokens
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

// f(token of the slice, place in the list) for the entries of a list of n that
// name the block's slice. `first` holds the thread's first four.
template <typename F>
__device__ __forceinline__ void rule_list(const uint32_t *list, uint32_t n, uint32_t base, u32x4a4 first, F f) {
    for (uint32_t i = threadIdx.x * 4; i < n; i += RULE_THREADS * 4) {
        if (i >= RULE_THREADS * 4) {
            if (i + 4 <= n) first = *(const u32x4a4 *)(list + i);
            else
#pragma unroll
                for (int e = 0; e < 4; e++) first[e] = i + e < n ? list[i + e] : 0;
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t t = first[e] - base;
            if (i + e < n && t < (uint32_t)RULE_SLICE) f(t, i + e);
        }
    }
}
__device__ __forceinline__ u32x4a4 rule_first(const uint32_t *list, uint32_t n) {
    const uint32_t i = threadIdx.x * 4;
    u32x4a4 x = {0, 0, 0, 0};
    if (i + 4 <= n) x = *(const u32x4a4 *)(list + i);
    else
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (i + e < n) x[e] = list[i + e];
    return x;
}

// Everything that a block reads is requested before the first wait: logits,
// mask words, the heads of the lists. The lists' tokens of the slice get a bit
// each, so that a thread asks once for its whole piece whether any rule names a
// value of it: nearly always none does, and the piece is masked and stored as
// loaded. `tables`: what the launch's rows need, 1 a count per token, 2 a bias
// per token (16 KB of LDS each).
template <int KIND>
__global__ __launch_bounds__(RULE_THREADS) void k_rules(RuleArgs a, RuleRows rr) {
    typedef RuleKind<KIND> K;
    typedef typename K::elem elem;
    constexpr int N = K::N, G = RULE_PER / N;
    extern __shared__ __align__(16) uint32_t tables[];
    __shared__ uint32_t named[RULE_SLICE / 32];
    __shared__ float best[RULE_THREADS / 64];
    __shared__ uint32_t first_at;
    const aotk_logits_rule r = rr.rule[blockIdx.y];
    const size_t row = (size_t)a.row0 + blockIdx.y;
    const uint32_t base = blockIdx.x * (uint32_t)RULE_SLICE;
    const int tid = threadIdx.x;
    const uint32_t left = a.vocab - base;  // tokens of the row from this slice on
    const elem *src = (const elem *)a.logits + row * a.stride + base;
    elem *dst = (elem *)a.out + row * a.stride + base;
    uint32_t *const cnt = tables, *const last = tables + (a.tables & 1 ? RULE_SLICE : 0);
    const bool pen = r.hist_len > 0 && (r.repetition != 1.0f || r.presence != 0.0f || r.frequency != 0.0f);
    const bool biased = r.bias_len > 0;

    u32x4 x[G];
    uint32_t word[G];
    const uint32_t *mask = r.mask >= 0 ? a.mask + (size_t)r.mask * ((a.vocab + 31) / 32) + base / 32 : nullptr;
#pragma unroll
    for (int g = 0; g < G; g++) {
        const uint32_t t = (g * RULE_THREADS + tid) * N;
        if (t + N <= left) {
            x[g] = *(const u32x4a2 *)(src + t);
        } else {  // the row ends inside the piece, or before it
            x[g] = u32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < N; i++)
                if (t + i < left) {
                    if constexpr (N == 4) x[g][i] = __float_as_uint(src[t + i]);
                    else x[g][i / 2] |= (uint32_t)src[t + i] << (i % 2 * 16);
                }
        }
        word[g] = mask && t < left ? mask[t / 32] >> (t % 32) : ~0u;
    }
    const u32x4a4 h0 = pen ? rule_first(a.hist + r.hist_off, r.hist_len) : u32x4a4{0, 0, 0, 0};
    const u32x4a4 b0 = biased ? rule_first(a.bias_id + r.bias_off, r.bias_len) : u32x4a4{0, 0, 0, 0};

    if (tid == 0) first_at = ~0u;
    if (pen || biased) {
        const u32x4 zero = {0, 0, 0, 0};
        for (int i = tid * 4; i < RULE_SLICE; i += RULE_THREADS * 4) {
            if (pen) *(u32x4 *)(cnt + i) = zero;
            if (biased) *(u32x4 *)(last + i) = zero;
        }
        if (tid < RULE_SLICE / 32) named[tid] = 0;
        __syncthreads();
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

    float top = -__builtin_inff();
#pragma unroll
    for (int g = 0; g < G; g++) {
        const uint32_t t = (g * RULE_THREADS + tid) * N;
        if (t >= left) continue;
        if (pen || biased) {
            const uint32_t who = (named[t / 32] >> (t % 32)) & ((1u << N) - 1);
            if (who)
#pragma unroll
                for (int i = 0; i < N; i++) {
                    if (!((who >> i) & 1u)) continue;
                    float v = K::get(x[g], i);
                    const uint32_t c = pen ? cnt[t + i] : 0, e = biased ? last[t + i] : 0;
                    if (c) v = (v > 0.0f ? v / r.repetition : v * r.repetition) - (r.presence + r.frequency * (float)c);
                    if (e) v = v + a.bias[(size_t)r.bias_off + e - 1];
                    K::set(x[g], i, v);
                }
        }
        uint32_t bits = word[g];
        if (t + N > left) bits &= (1u << (left - t)) - 1;  // nothing behind the row's end is picked
        if (mask || t + N > left) K::allow(x[g], bits);
        if (t + N <= left) {
            *(u32x4a2 *)(dst + t) = x[g];
        } else {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (t + i < left) {
                    if constexpr (N == 4) dst[t + i] = __uint_as_float(x[g][i]);
                    else dst[t + i] = (uint16_t)(x[g][i / 2] >> (i % 2 * 16));
                }
        }
        if (a.keys)  // NaN is passed over
#pragma unroll
            for (int i = 0; i < N; i++) top = fmaxf(top, K::get(x[g], i));
    }
    if (!a.keys) return;
    float most = top;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, shfl_xor(most, o));
    if ((tid & 63) == 0) best[tid >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < RULE_THREADS / 64; w++) most = fmaxf(most, best[w]);
    if (top == most && most > -__builtin_inff()) {  // whoever holds it: the lowest token
#pragma unroll
        for (int g = G - 1; g >= 0; g--)
#pragma unroll
            for (int i = N - 1; i >= 0; i--) {
                const uint32_t t = (g * RULE_THREADS + tid) * N + i;
                if (t < left && K::get(x[g], i) == most) atomicMin(&first_at, t);
            }
    }
    __syncthreads();
    if (tid == 0) a.keys[row * gridDim.x + blockIdx.x] = first_at == ~0u ? 0 : rule_key(most, base + first_at);
}

// One wave per row: the best of its slices' keys.
__global__ __launch_bounds__(64) void k_rules_pick(const uint64_t *keys, int n, uint32_t *tokens) {
    uint64_t k = 0;
    for (int i = threadIdx.x; i < n; i += 64) {
        const uint64_t o = keys[(size_t)blockIdx.x * n + i];
        k = o > k ? o : k;
    }
    k = wave_max_key(k);
    if (threadIdx.x == 0) tokens[blockIdx.x] = k ? ~(uint32_t)k : 0xFFFFFFFFu;
}

size_t rules_scratch_bytes(size_t rows, size_t vocab) { return rows * ((vocab + RULE_SLICE - 1) / RULE_SLICE) * 8; }

void launch_rules(int kind, RuleArgs a, const aotk_logits_rule *rules, size_t rows, uint32_t *tokens, hipStream_t s) {
    const unsigned slices = (a.vocab + RULE_SLICE - 1) / RULE_SLICE;
    RuleRows rr;
    for (size_t r0 = 0; r0 < rows; r0 += RULE_ROWS) {
        const size_t n = rows - r0 < (size_t)RULE_ROWS ? rows - r0 : (size_t)RULE_ROWS;
        for (size_t i = 0; i < n; i++) rr.rule[i] = rules[r0 + i];
        for (size_t i = n; i < (size_t)RULE_ROWS; i++) rr.rule[i] = aotk_logits_rule{};
        a.row0 = (uint32_t)r0;
        a.tables = 0;
        for (size_t i = 0; i < n; i++) a.tables |= (rr.rule[i].hist_len ? 1u : 0u) | (rr.rule[i].bias_len ? 2u : 0u);
        const size_t lds = ((a.tables & 1) + (a.tables >> 1)) * RULE_SLICE * sizeof(uint32_t);
        const dim3 grid(slices, (unsigned)n);
        switch (kind) {
        case AOTK_F32: k_rules<AOTK_F32><<<grid, RULE_THREADS, lds, s>>>(a, rr); break;
        case AOTK_F16: k_rules<AOTK_F16><<<grid, RULE_THREADS, lds, s>>>(a, rr); break;
        default: k_rules<AOTK_BF16><<<grid, RULE_THREADS, lds, s>>>(a, rr); break;
        }
    }
    if (tokens) k_rules_pick<<<(unsigned)rows, 64, 0, s>>>(a.keys, (int)slices, tokens);
}

}  // namespace aotk
