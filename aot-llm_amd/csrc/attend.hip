// attend.hip - attention over two ranges of keys, in the caches' own type
// (f32, f16, bf16): rows that see a sliding window and the first positions of
// their sequence, and rows of a batch of sequences that share one prefix.
//
// Row i of sequence b sees all of the shared range and, of the sequence's own
// range, the positions j <= p(i) with j < n_sink, window == 0 or j > p(i) - window:
//   s_j = <q, k_j> / sqrt(D),  o = sum_j e^(s_j - max) v_j / sum_j e^(s_j - max)
// Scores, exponents, sums and the output's accumulation are f32; the output is
// rounded once to the caches' type. A row that sees nothing is 0.
#include "device.hpp"
#include "internal.hpp"

namespace aotk {

template <int KIND>
struct AttElem;
template <>
struct AttElem<AOTK_F32> {
    typedef float elem;
    static __device__ __forceinline__ float up(float x) { return x; }
    static __device__ __forceinline__ float down(float x) { return x; }
};
template <>
struct AttElem<AOTK_F16> {
    typedef uint16_t elem;
    static __device__ __forceinline__ float up(uint16_t x) { return f16_to_f32(x); }
    static __device__ __forceinline__ uint16_t down(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};
template <>
struct AttElem<AOTK_BF16> {
    typedef uint16_t elem;
    static __device__ __forceinline__ float up(uint16_t x) { return bf16_to_f32(x); }
    static __device__ __forceinline__ uint16_t down(float x) { return f32_to_bf16(x); }
};

// One wave per (row, query head), the keys one after another.
template <int KIND, int D>
__global__ __launch_bounds__(64) void k_attend_plain(AttendArgs a, AttendSeqs sq) {
    typedef AttElem<KIND> E;
    typedef typename E::elem elem;
    constexpr int N = D / 64;
    const int h = blockIdx.x, lane = threadIdx.x;
    const AttendSeq s = sq.seq[blockIdx.z];
    const uint32_t i = blockIdx.y;
    if (i >= s.rows) return;
    const size_t kvh = h / (a.n_head / a.n_kv_head), kv = (size_t)a.n_kv_head * D;
    const size_t at = ((size_t)(s.row0 + i) * a.n_head + h) * D + lane;
    float q[N], acc[N];
#pragma unroll
    for (int e = 0; e < N; e++) {
        q[e] = E::up(((const elem *)a.q)[at + e * 64]);
        acc[e] = 0.0f;
    }
    float mx = -__builtin_inff(), sum = 0.0f;
    auto key = [&](const elem *k, const elem *v) {
        float d = 0.0f;
#pragma unroll
        for (int e = 0; e < N; e++) d += q[e] * E::up(k[lane + e * 64]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) d += shfl_xor(d, o);
        d *= a.scale;
        const float m2 = fmaxf(mx, d), base = m2 == -__builtin_inff() ? 0.0f : m2;
        const float c = __expf(mx - base), p = __expf(d - base);
        sum = sum * c + p;
#pragma unroll
        for (int e = 0; e < N; e++) acc[e] = acc[e] * c + p * E::up(v[lane + e * 64]);
        mx = m2;
    };
    for (size_t j = 0; j < a.n_prefix; j++)
        key((const elem *)a.k_prefix + j * kv + kvh * D, (const elem *)a.v_prefix + j * kv + kvh * D);
    const int64_t p = (int64_t)s.len - s.rows + i;  // the row's position in its own range
    const size_t own = s.cache * kv;
    bool any = a.n_prefix > 0;
    for (int64_t j = 0; j <= p; j++) {
        if (a.window && j >= (int64_t)a.n_sink && j <= p - (int64_t)a.window) continue;
        any = true;
        key((const elem *)a.k + own + j * kv + kvh * D, (const elem *)a.v + own + j * kv + kvh * D);
    }
#pragma unroll
    for (int e = 0; e < N; e++) ((elem *)a.out)[at + e * 64] = E::down(any ? acc[e] / sum : 0.0f);
}

size_t attend_scratch_bytes(const AttendArgs &, const AttendSeq *, size_t) { return 0; }

void launch_attend(int kind, int head_dim, const AttendArgs &a, const AttendSeq *seqs, size_t n, void *, hipStream_t s) {
    AttendSeqs sq = {};
    for (size_t b0 = 0; b0 < n; b0 += ATTEND_SEQS) {
        const size_t nb = n - b0 < (size_t)ATTEND_SEQS ? n - b0 : (size_t)ATTEND_SEQS;
        uint32_t most = 0;
        for (size_t i = 0; i < nb; i++) {
            sq.seq[i] = seqs[b0 + i];
            most = most > seqs[b0 + i].rows ? most : seqs[b0 + i].rows;
        }
        if (!most) continue;
        const dim3 grid((unsigned)a.n_head, most, (unsigned)nb);
#define L(K, D) k_attend_plain<K, D><<<grid, 64, 0, s>>>(a, sq)
#define K(D) (kind == AOTK_F32 ? L(AOTK_F32, D) : kind == AOTK_F16 ? L(AOTK_F16, D) : L(AOTK_BF16, D))
        if (head_dim == 64) K(64);
        else if (head_dim == 128) K(128);
        else K(256);
#undef K
#undef L
    }
}

}  // namespace aotk
