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
template <bool FAST>
__device__ __forceinline__ float gated_act(int act, float g)
{
    switch (act) {
    case PT_GATE_SILU: return g * gated_sigmoid<FAST>(g);
    case PT_GATE_GELU: return g * (0.5f * (1.0f + erff(g * 0.707106781f)));
    case PT_GATE_RELU: return g > 0.0f || g != g ? g : 0.0f;
    default: return gated_sigmoid<FAST>(g);
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
        const float below = 0.5f * (1.0f + erff(g * 0.707106781f));
        const float bell = FAST ? __builtin_amdgcn_exp2f(g * g * -0.72134752f) : expf(-0.5f * g * g);
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
        slope = s * (1.0f - s);
    }
    }
}

// What a pair of products is stored as: act(P0) P1, that and both products
// (for the gradient), both products, or fp32 parts of a split contraction.
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
    int act;
    int tiles_m, tiles_n, split, stages;  // stages: 64-wide K stages of a split's share
};
constexpr long long kPairPitch = 1 << 21;  // the most that a row's pitch may be

void pair_plan(PairArgs &g, bool columns, int &tm);  // tiles, split and stages
void launch_pair_columns(const PairArgs &g, int dtype, int tm, int store, hipStream_t s);
void launch_pair_sum(const PairArgs &g, int dtype, int tm, hipStream_t s);
// the join alone: of few rows' parts, columns form (also float32)
void launch_pair_join(const PairArgs &g, int dtype, int store, hipStream_t s);

}  // namespace pt
