// Internal header of the gated projection (pt_gated.hip, pt_gated_ring.hip).
// Not part of the public boundary (include/pt_hip.h is).
#pragma once

#include "pt_gemm.h"

namespace pt {

// act(g) and its derivative.  FAST (16-bit results): the hardware's 2^x and
// reciprocal, each within an ulp; 2^(-g log2 e) is then off by |g| 2^-24 of
// itself, far below the result's rounding.
template <bool FAST>
__device__ __forceinline__ float gated_sigmoid(float g)
{
    if constexpr (FAST) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504f));
    else return 1.0f / (1.0f + expf(-g));
}
// The standard normal's distribution and exp(-g^2 / 2), by erfc, so that the
// small values of negative g keep their digits (1 + erf has none left below
// -6).  FAST: erfc(z) = e^(-z^2) t Q(t) with t = 1 / (1 + 0.44 z), Q fitted to
// the least relative error, 1.9e-7 for z >= 0.
template <bool FAST>
__device__ __forceinline__ float gated_below(float g, float &bell)
{
    if constexpr (!FAST) {
        bell = expf(-0.5f * g * g);
        return 0.5f * erfcf(g * -0.707106781f);
    } else {
        bell = __builtin_amdgcn_exp2f(g * g * -0.72134752f);
        const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(g), 0.44f * 0.707106781f, 1.0f));
        float q = fmaf(t, 0.07150499f, -0.27917263f);
        q = fmaf(t, q, 0.29889796f);
        q = fmaf(t, q, -0.02231892f);
        q = fmaf(t, q, 0.21700441f);
        q = fmaf(t, q, 0.21693216f);
        q = fmaf(t, q, 0.2489357f);
        q = fmaf(t, q, 0.24821652f);
        const float tail = 0.5f * q * t * bell;
        return g < 0.0f ? tail : 1.0f - tail;
    }
}
template <bool FAST>
__device__ __forceinline__ float gated_act(int act, float g)
{
    float bell;
    switch (act) {
    case PT_GATE_SILU: return g * gated_sigmoid<FAST>(g);
    case PT_GATE_GELU: return g * gated_below<FAST>(g, bell);
    case PT_GATE_RELU: return g > 0.0f || g != g ? g : 0.0f;
    default: return gated_sigmoid<FAST>(g);
    }
}
// p = act(p) q for N of them: one branch, and little code for the
// instruction cache, which a short kernel finds empty
template <bool FAST, int N>
__device__ __forceinline__ void gated_products(int act, float (&p)[N], const float (&q)[N])
{
    auto all = [&](auto ACT) {
#pragma unroll
        for (int k = 0; k < N; k++) p[k] = gated_act<FAST>(decltype(ACT)::value, p[k]) * q[k];
    };
    switch (act) {
    case PT_GATE_SILU: return all(IC<PT_GATE_SILU>{});
    case PT_GATE_GELU: return all(IC<PT_GATE_GELU>{});
    case PT_GATE_RELU: return all(IC<PT_GATE_RELU>{});
    default: return all(IC<PT_GATE_SIGMOID>{});
    }
}
template <bool FAST>
__device__ __forceinline__ void gated_slope(int act, float g, float &value, float &slope)
{
    switch (act) {
    case PT_GATE_SILU: {
        const float s = gated_sigmoid<FAST>(g);
        value = g * s;
        slope = s * (1.0f + g * (1.0f - s));
        break;
    }
    case PT_GATE_GELU: {
        float bell;
        const float below = gated_below<FAST>(g, bell);
        value = g * below;
        slope = below + g * bell * 0.398942280f;
        break;
    }
    case PT_GATE_RELU:
        value = g > 0.0f || g != g ? g : 0.0f;
        slope = g > 0.0f ? 1.0f : 0.0f;
        break;
    default: {
        const float s = gated_sigmoid<FAST>(g);
        value = s;
        slope = s * gated_sigmoid<FAST>(-g);  // (1 - s has no digits left where g is large)
    }
    }
}

// What the gradient keeps of a product of 16-bit operands: its float32 value's
// upper 24 bits, 16 of them in one plane and 8 in another.  Rounded to the
// operands' type instead, both products' errors would come on top of those
// of dg and du: gradients off by 1.8 times a result's own rounding instead
// of 1.4, for 4 bytes an element instead of 6.
__device__ __forceinline__ uint32_t kept_high(float v) { return __float_as_uint(v) >> 16; }
__device__ __forceinline__ uint32_t kept_low(float v) { return __float_as_uint(v) >> 8 & 0xffu; }
__device__ __forceinline__ float kept_value(uint32_t high, uint32_t low) { return __uint_as_float(high << 16 | low << 8); }
// where the planes of the two products of n elements lie, high and low
__device__ __host__ __forceinline__ long long kept_plane(long long n, int product, bool low) { return low ? 4 * n + product * n : 2 * n * product; }

// One element of both products, as the gradient keeps them: float32 beside
// each other's planes, or in 24 bits.
template <int DT>
__device__ __forceinline__ void gated_keep(void *kept, long long n, long long i, float p, float q)
{
    if constexpr (DT == PT_FLOAT32) {
        ((float *)kept)[i] = p;
        ((float *)kept)[n + i] = q;
    } else {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            ((uint16_t *)((char *)kept + kept_plane(n, k, false)))[i] = (uint16_t)kept_high(k ? q : p);
            ((uint8_t *)kept + kept_plane(n, k, true))[i] = (uint8_t)kept_low(k ? q : p);
        }
    }
}

// float16 gradients: dg and du leave float16's range where their products with
// the operands do not (an upstream gradient of a mean, a large product), so
// they are multiplied by powers of two that take the largest of a row (for
// dx) or of a column (for dgate and dup) into [2^14, 2^15), and the sums are
// multiplied back in float32.  What is below 2^-29 of that largest one has
// fewer than float16's digits, within 2^-39 of it.  (bfloat16 has float32's
// range.)  Shifts past these bounds change no float16 result.
__device__ __forceinline__ int gated_shift(float top)
{
    return top > 0.0f ? min(14 + 127 - (int)(__float_as_uint(top) >> 23), 100) : 0;
}

// What a pair of products is stored as: act(P0) P1, that and both products as
// the gradient keeps them (c1), both products (c1, c2), or fp32 parts of a
// split contraction.
enum { GATED_PRODUCT = 0, GATED_KEPT = 1, GATED_BOTH = 2, GATED_PARTS = 3 };

// Products over a pair of matrices, 16 bits (pt_gated_ring.hip).
//   launch_pair_columns: P0 = A B0 and P1 = A B1; A [M][K], B [K][N].
//   launch_pair_sum: P = A0 B0^T + A1 B1^T; A [M][K], B [N][K].
// Rows start at 16-byte boundaries (pitches lda, ldb multiples of 8).
struct PairArgs {
    const void *a0, *a1, *b0, *b1;
    long long lda, ldb;
    int M, N, K;     // K a multiple of 8: past its end A's rows are not read ..
    int kb;          // .. nor B's rows from kb <= K on (columns form); zeros instead
    int n_out;       // columns that are stored (columns form: N is a multiple of 8)
    void *c0, *c1, *c2;  // results, contiguous
    float *parts;    // [split][1 or 2][M][n_out]
    const int8_t *shift;  // float16 gradients: the power of two that A's row (sum form, [M]) or B's column (columns form,
                          // of both matrices, [2][n_out]) was multiplied by
    int act;
    int tiles_m, tiles_n, split, stages;  // stages: 64-wide K stages of a split's share
};
constexpr long long kPairPitch = 1 << 21;  // the most that a row's pitch may be

void pair_plan(PairArgs &g, bool columns, int &tm);  // tiles, split and stages
void launch_pair_columns(const PairArgs &g, int dtype, int tm, int store, hipStream_t s);
void launch_pair_sum(const PairArgs &g, int dtype, int tm, hipStream_t s);
// the join alone, of parts that were made elsewhere: float32, and few rows in
// the columns form
void launch_pair_join(const PairArgs &g, int dtype, bool sum, int store, hipStream_t s);

// The same of fp32 matrices at any pitch (pt_gated_wide.hip): kb is not read,
// stages are 16 k wide; turned: columns with A [K][M].
enum { WIDE_COLUMNS = 0, WIDE_TURNED = 1, WIDE_SUM = 2 };
void wide_plan(PairArgs &g, int form, int &tm);
void launch_wide(const PairArgs &g, int tm, int form, int store, hipStream_t s);

}  // namespace pt
