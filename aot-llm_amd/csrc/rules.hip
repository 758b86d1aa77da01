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

constexpr int RULE_THREADS = 256;
constexpr int RULE_PER = RULE_SLICE / RULE_THREADS;  // values per thread

// Rows start at any multiple of the element size: vector accesses that
// promise no more alignment than that.
template <int KIND>
struct RuleVec;
template <>
struct RuleVec<AOTK_F32> {
    typedef float elem;
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
    static constexpr int N = 4;
    static __device__ __forceinline__ float up(float x) { return x; }
    static __device__ __forceinline__ float down(float x) { return x; }
};
template <>
struct RuleVec<AOTK_F16> {
    typedef uint16_t elem;
    typedef uint16_t vec __attribute__((ext_vector_type(8), aligned(2)));
    static constexpr int N = 8;
    static __device__ __forceinline__ float up(uint16_t x) { return f16_to_f32(x); }
    // one conversion, to nearest even (overflow to infinity)
    static __device__ __forceinline__ uint16_t down(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};
template <>
struct RuleVec<AOTK_BF16> {
    typedef uint16_t elem;
    typedef uint16_t vec __attribute__((ext_vector_type(8), aligned(2)));
    static constexpr int N = 8;
    static __device__ __forceinline__ float up(uint16_t x) { return bf16_to_f32(x); }
    static __device__ __forceinline__ uint16_t down(float x) { return f32_to_bf16(x); }
};

// Pick key: the value's order in the high word, the complement of the token
// in the low one (the maximum is the largest value's lowest token). 0 stands
// for no token: NaN and -inf are never picked. Zeros of both signs are equal.
__device__ __forceinline__ uint64_t rule_key(float y, uint32_t t) {
    if (!(y > -__builtin_inff())) return 0;
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

template <int KIND>
__global__ __launch_bounds__(RULE_THREADS) void k_rules(RuleArgs a, RuleRows rr) {
    typedef RuleVec<KIND> VT;
    typedef typename VT::elem elem;
    typedef typename VT::vec vec;
    constexpr int N = VT::N, G = RULE_PER / N;
    __shared__ uint32_t cnt[RULE_SLICE];
    __shared__ uint32_t last[RULE_SLICE];
    __shared__ uint64_t best[RULE_THREADS / 64];
    const aotk_logits_rule r = rr.rule[blockIdx.y];
    const size_t row = (size_t)a.row0 + blockIdx.y;
    const uint32_t base = blockIdx.x * (uint32_t)RULE_SLICE;
    const int tid = threadIdx.x;
    const uint32_t left = a.vocab - base;  // tokens of the row from this slice on
    const elem *src = (const elem *)a.logits + row * a.stride + base;
    elem *dst = (elem *)a.out + row * a.stride + base;

    // the slice's logits, in flight while the lists are scanned
    vec x[G];
#pragma unroll
    for (int g = 0; g < G; g++) {
        const uint32_t t = (g * RULE_THREADS + tid) * N;
        if (t + N <= left) x[g] = *(const vec *)(src + t);
        else
#pragma unroll
            for (int i = 0; i < N; i++) x[g][i] = t + i < left ? src[t + i] : (elem)0;
    }

    const bool pen = r.hist_len > 0 && (r.repetition != 1.0f || r.presence != 0.0f || r.frequency != 0.0f);
    const bool biased = r.bias_len > 0;
    if (pen || biased) {
        for (int i = tid; i < RULE_SLICE; i += RULE_THREADS) {
            cnt[i] = 0;
            last[i] = 0;
        }
        __syncthreads();
        if (pen)
            for (uint32_t i = tid; i < r.hist_len; i += RULE_THREADS) {
                const uint32_t t = a.hist[(size_t)r.hist_off + i] - base;
                if (t < (uint32_t)RULE_SLICE) atomicAdd(&cnt[t], 1u);
            }
        if (biased)
            for (uint32_t i = tid; i < r.bias_len; i += RULE_THREADS) {
                const uint32_t t = a.bias_id[(size_t)r.bias_off + i] - base;
                if (t < (uint32_t)RULE_SLICE) atomicMax(&last[t], i + 1);
            }
        __syncthreads();
    }
    const uint32_t *mask = r.mask >= 0 ? a.mask + (size_t)r.mask * ((a.vocab + 31) / 32) + base / 32 : nullptr;

    uint64_t key = 0;
#pragma unroll
    for (int g = 0; g < G; g++) {
        const uint32_t t = (g * RULE_THREADS + tid) * N;
        if (t >= left) continue;
        const uint32_t word = mask ? mask[t / 32] >> (t % 32) : ~0u;
        vec y;
#pragma unroll
        for (int i = 0; i < N; i++) {
            float v = VT::up(x[g][i]);
            if (pen) {
                const uint32_t c = cnt[t + i];
                if (c) v = (v > 0.0f ? v / r.repetition : v * r.repetition) - (r.presence + r.frequency * (float)c);
            }
            if (biased) {
                const uint32_t e = last[t + i];
                if (e) v = v + a.bias[(size_t)r.bias_off + e - 1];
            }
            if (!((word >> i) & 1u)) v = -__builtin_inff();
            y[i] = VT::down(v);
            const uint64_t k = t + i < left ? rule_key(VT::up(y[i]), base + t + i) : 0;
            key = k > key ? k : key;
        }
        if (t + N <= left) *(vec *)(dst + t) = y;
        else
#pragma unroll
            for (int i = 0; i < N; i++)
                if (t + i < left) dst[t + i] = y[i];
    }
    if (!a.keys) return;
    key = wave_max_key(key);
    if ((tid & 63) == 0) best[tid >> 6] = key;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < RULE_THREADS / 64; w++) key = best[w] > key ? best[w] : key;
        a.keys[row * gridDim.x + blockIdx.x] = key;
    }
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
        const dim3 grid(slices, (unsigned)n);
        switch (kind) {
        case AOTK_F32: k_rules<AOTK_F32><<<grid, RULE_THREADS, 0, s>>>(a, rr); break;
        case AOTK_F16: k_rules<AOTK_F16><<<grid, RULE_THREADS, 0, s>>>(a, rr); break;
        default: k_rules<AOTK_BF16><<<grid, RULE_THREADS, 0, s>>>(a, rr); break;
        }
    }
    if (tokens) k_rules_pick<<<(unsigned)rows, 64, 0, s>>>(a.keys, (int)slices, tokens);
}

}  // namespace aotk
