// Attention kernels for gfx950: forward, gradients of keys and values, and
// gradient of queries, as templates over the element type and the padded
// head size.  Instantiated per type in pt_attention_{bf16,f16,f32}.hip and
// launched by pt_attention.hip.  Not part of the public boundary.
//
// For query i and key j of one sequence and head, with c = scale:
//   s_ij = c q_i . k_j            over the keys that i sees
//   o_i  = sum_j p_ij v_j,        p_ij = exp(s_ij - lse_i)
//   lse_i = log sum_j exp(s_ij)
// and, for the upstream gradient w_i of o_i,
//   d_i = w_i . o_i,  t_ij = p_ij (w_i . v_j - d_i)
//   dv_j = sum_i p_ij w_i,  dk_j = c sum_i t_ij q_i,  dq_i = c sum_j t_ij k_j
//
// Every product runs on 32x32 MFMA blocks whose column (lane % 32) is the
// row that stays in the wave: a query in the forward pass and in the
// queries' gradient, a key in the keys' and values'.  The block's rows are
// then the streamed side, and a lane holds 16 of its column's 32 values
// (row 8 (r / 4) + 4 (lane / 32) + r % 4 in register r), so a softmax row is
// reduced inside two lanes.  Those registers are already the second
// product's right operand: the product sums over the streamed rows in any
// order, so its k slots are numbered the way the registers hold them, and
// the left operand is read from LDS in that same order.  Probabilities
// never pass through LDS.
#pragma once

#include <limits.h>

#include "pt_gemm.h"

namespace pt {

struct AttnArgs {
    const void *q, *k, *v;
    void *out;
    float *lse;
    // strides in elements: sequence (0 where starts are given), token, head
    long long q_bs, q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs, o_bs, o_ts, o_hs;
    const int32_t *q_starts, *q_lengths, *k_starts, *k_lengths;  // device, or null
    int batch, heads, kv_heads, group, size, nq, nk, q_rows, k_rows;
    int causal;
    float scale, scale_log2;
    int splits;               // key ranges computed by workgroups of their own
    float *part_o, *part_ml;  // their results: [split][sequence, key head][row][size], and (m, l)
    // backward
    const void *w;            // upstream gradient in the element type, contiguous like out
    const float *lse2, *delta;  // per (head, token row): lse in base 2 (+inf where nothing is seen), d
    void *dq, *dk, *dv;
    long long stat_rows;      // token rows of a head in lse, lse2 and delta
};

struct AttnSeq {
    long long row;  // first token row in a packed tensor
    int n;          // tokens
};

// What the device arrays say of sequence b, held inside the tensor whatever
// they say.
__device__ __forceinline__ AttnSeq attn_seq(const int32_t *starts, const int32_t *lengths, int rows, int most, int b)
{
    if (!starts) return {0, most};
    const int s = min(max(starts[b], 0), rows);
    return {s, min(max(lengths[b], 0), min(most, rows - s))};
}

template <int DT> struct AttnT {
    using S = typename GE<DT>::S;
    using Frag = typename FragT<DT>::type;
    static constexpr int PK = GE<DT>::PK;  // elements of a 16-byte chunk
    static constexpr int ES = (int)sizeof(S);
};

// A staged tile keeps its rows whole, the 16-byte chunks of row r permuted
// by an exclusive or.  A row read takes one chunk of 16 consecutive rows, a
// transposing read 64 bytes of 4 consecutive rows; with 16 or more chunks
// to a row the low two bits of r therefore move groups of four chunks and
// the next two move chunks inside a group, so both touch every bank once.
template <int CPR>
__device__ __forceinline__ int attn_swz(int r)
{
    if constexpr (CPR >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    else return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

// Source of the rows of one sequence and head.
struct AttnSrc {
    const char *base;  // row 0
    long long step;    // bytes from row to row
    int rows;
};

// The byte offsets of a lane's chunks in a tile, for chunks that may be
// loaded as 16 bytes (VEC), relative to the tile's first row.
template <int DT, int DP, int ROWS, int NW, bool VEC> struct AttnStage {
    using T = AttnT<DT>;
    using S = typename T::S;
    static constexpr int CPR = DP * T::ES / 16;
    static constexpr int NI = ROWS * CPR / 64 / NW;  // 1 KiB instructions of each wave
    static_assert(ROWS * CPR == NI * 64 * NW, "whole instructions");
    uint32_t off[VEC ? NI : 1];

    __device__ __forceinline__ void init(const AttnSrc &s, int size, int wave, int lane)
    {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int at = (wave * NI + i) * 64 + lane, row = at / CPR, c = (at % CPR) ^ attn_swz<CPR>(row);
                // past the head's size: past every range, read as zero
                off[i] = c * T::PK < size ? (uint32_t)(row * s.step) + (uint32_t)c * 16u : 0xfffffff0u;
            }
        }
    }
    // Rows r0 .. r0 + ROWS - 1 into `tile`; rows past the source's last are zeros.
    __device__ __forceinline__ void load(const AttnSrc &s, int size, int r0, S *tile, int wave, int lane) const
    {
        const char *base = s.base + (long long)r0 * s.step;
        if constexpr (VEC) {
            const long long left = (long long)(s.rows - r0 - 1) * s.step + size * T::ES;
            const uint32_t range = r0 >= s.rows ? 0u : (uint32_t)min(left, (long long)0x7fffffff);
#pragma unroll
            for (int i = 0; i < NI; i++)
                buffer_load_lds16(base, off[i], (PT_LDS_AS void *)(tile + (wave * NI + i) * 64 * T::PK), range);
        } else {
            for (int i = 0; i < NI; i++) {
                const int at = (wave * NI + i) * 64 + lane, row = at / CPR, c = (at % CPR) ^ attn_swz<CPR>(row);
                alignas(16) S e[T::PK];
#pragma unroll
                for (int x = 0; x < T::PK; x++) {
                    const int d = c * T::PK + x;
                    e[x] = r0 + row < s.rows && d < size ? ((const S *)(base + (long long)row * s.step))[d] : (S)0;
                }
                *(floatx4 *)(tile + at * T::PK) = *(const floatx4 *)e;
            }
        }
    }
};

// One lane's row as the right operand of the products over the head's size:
// fragment t holds chunk 2 t + lane / 32.
template <int DT, int DP, bool VEC>
__device__ __forceinline__ void attn_row(typename AttnT<DT>::Frag (&f)[DP * AttnT<DT>::ES / 32], const void *row, bool live,
                                         int size, int half)
{
    using T = AttnT<DT>;
    using S = typename T::S;
#pragma unroll
    for (int t = 0; t < DP * T::ES / 32; t++) {
        const int d = (2 * t + half) * T::PK;
        floatx4 raw = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (VEC) {
            if (live && d < size) raw = *(const floatx4 *)((const S *)row + d);
        } else if (live) {
            alignas(16) S e[T::PK];
#pragma unroll
            for (int x = 0; x < T::PK; x++) e[x] = d + x < size ? ((const S *)row)[d + x] : (S)0;
            raw = *(const floatx4 *)e;
        }
        f[t] = __builtin_bit_cast(typename T::Frag, raw);
    }
}

template <int DT>
__device__ __forceinline__ void attn_mfma(floatx16 &acc, const typename AttnT<DT>::Frag &a,
                                          const typename AttnT<DT>::Frag &b)
{
    if constexpr (DT == PT_FLOAT32) {
#pragma unroll
        for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], acc, 0, 0, 0);
    } else if constexpr (DT == PT_BFLOAT16) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
    } else {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
    }
}

// A lane's byte offsets into a staged tile: of its row's chunk in a row read,
// and of its pieces in the two transposing reads (16-bit) or of its element
// (float32).  The chunk that step t or element block d takes is the base's
// with t or d in other bits, put in by an exclusive or at the read: three
// registers serve every read of every tile.  `fresh` keeps the compiler from
// computing all the addresses ahead of the loop, which spilled registers.
template <int DT, int DP> struct AttnLane {
    static constexpr int ES = AttnT<DT>::ES, CPR = DP * ES / 16;
    uint32_t row, col0, col1;

    __device__ __forceinline__ void init(int lane)
    {
        const int half = lane >> 5, r = lane & 31;
        row = (uint32_t)(r * DP * ES + ((half ^ attn_swz<CPR>(r)) << 4));
        if constexpr (DT == PT_FLOAT32) {
            col0 = col1 = (uint32_t)(4 * half * DP * 4 + (((r >> 2) ^ (half & 3)) << 4) + (r & 3) * 4);
        } else {
            const int s = lane & 15, c = ((lane >> 4) & 1) * 2 + ((s & 3) >> 1), r0 = 4 * half + (s >> 2), r1 = r0 + 8;
            col0 = (uint32_t)(r0 * DP * ES + ((c ^ attn_swz<CPR>(r0)) << 4) + (s & 1) * 8);
            col1 = (uint32_t)(r1 * DP * ES + ((c ^ attn_swz<CPR>(r1)) << 4) + (s & 1) * 8);
        }
    }
    __device__ __forceinline__ void fresh() { asm volatile("" : "+v"(row), "+v"(col0), "+v"(col1)); }
};

// acc[streamed row][own row] = sum over the head's size, for the 32 tile
// rows from row0.
template <int DT, int DP>
__device__ __forceinline__ floatx16 attn_rows(const typename AttnT<DT>::S *tile, int row0,
                                              const typename AttnT<DT>::Frag (&b)[DP * AttnT<DT>::ES / 32],
                                              const AttnLane<DT, DP> &at)
{
    using T = AttnT<DT>;
    floatx16 acc;
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] = 0.0f;
    const PT_LDS_AS char *base = (const PT_LDS_AS char *)tile + row0 * DP * T::ES;
#pragma unroll
    for (int t = 0; t < DP * T::ES / 32; t++) {
        const floatx4 a = *(const PT_LDS_AS floatx4 *)(base + (at.row ^ (uint32_t)(t << 5)));
        attn_mfma<DT>(acc, __builtin_bit_cast(typename T::Frag, a), b[t]);
    }
    return acc;
}

typedef float attn_f32x2 __attribute__((ext_vector_type(2)));
typedef float attn_f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 attn_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 attn_f16x8 __attribute__((ext_vector_type(8)));

// Registers 8 u .. 8 u + 7 of a block rounded to the element type: the right
// operand of the product over the streamed rows.
template <int DT>
__device__ __forceinline__ typename AttnT<DT>::Frag attn_pack(const floatx16 &p, int u)
{
    attn_f32x8 v;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = p[8 * u + i];
    if constexpr (DT == PT_BFLOAT16) return __builtin_convertvector(v, attn_bf16x8);
    else return __builtin_convertvector(v, attn_f16x8);
}

// acc[x] += (32 tile rows from row0)^T p, where p holds a block's registers:
// acc[x] is [32 x + element of the head][own row].
//
// 16-bit: a transposing read gives lane s of 16 the s-th of 16 columns in 4
// rows; two of them fill the 8 k slots, rows 4 half + 0..3 and 8 + 4 half +
// 0..3, which are the rows that registers 8 u .. 8 u + 7 hold.  float32: one
// k slot for each half of the wave, register r's row.
template <int DT, int DP>
__device__ __forceinline__ void attn_cols(floatx16 (&acc)[DP / 32], const typename AttnT<DT>::S *tile, int row0,
                                          const floatx16 &p, const AttnLane<DT, DP> &at)
{
    using T = AttnT<DT>;
    const PT_LDS_AS char *base = (const PT_LDS_AS char *)tile + row0 * DP * T::ES;
    if constexpr (DT == PT_FLOAT32) {
#pragma unroll
        for (int r = 0; r < 16; r++) {
            // rows 8 (r / 4) + r % 4 (+ 4 half): the swizzle's bits of r, the half's are in the base
            const int x = (r % 4) << 2 | ((r / 4) * 2 & 3);
#pragma unroll
            for (int d = 0; d < DP / 32; d++) {
                const float a = *(const PT_LDS_AS float *)(base + (8 * (r / 4) + r % 4) * DP * 4 +
                                                           (at.col0 ^ (uint32_t)((8 * d ^ x) << 4)));
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[r], acc[d], 0, 0, 0);
            }
        }
    } else {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const typename T::Frag b = attn_pack<DT>(p, u);
#pragma unroll
            for (int d = 0; d < DP / 32; d++) {
                typedef short v4s __attribute__((ext_vector_type(4)));
                const PT_LDS_AS char *to = base + u * 16 * DP * T::ES;
                const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((PT_LDS_AS v4s *)(to + (at.col0 ^ (uint32_t)(d << 6))));
                const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((PT_LDS_AS v4s *)(to + (at.col1 ^ (uint32_t)(d << 6))));
                const auto a = __builtin_bit_cast(typename T::Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                attn_mfma<DT>(acc[d], a, b);
            }
        }
    }
}

// Everything this wave loads or writes to LDS is there, and every wave has
// come here: the loads to LDS are waited for by hand, since the compiler's
// own barrier need not wait for them.
__device__ __forceinline__ void attn_landed()
{
    ring_wait<0>();
    ring_barrier();
}

// The other half's value of the same column.
__device__ __forceinline__ float attn_other(float v, int lane)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(lane < 32 ? r[1] : r[0]);
}

// Four consecutive elements of a contiguous row from e on, where e + 4 may
// pass the head's size; ALIGNED: the size is a multiple of four.
template <int DT>
__device__ __forceinline__ void attn_store4(void *row, int e, int size, float a, float b, float c, float d)
{
    using S = typename AttnT<DT>::S;
    if (e >= size) return;
    S *p = (S *)row + e;
    const float v[4] = {a, b, c, d};
    if ((size & 3) == 0) {
        if constexpr (DT == PT_FLOAT32) {
            *(floatx4 *)p = floatx4{a, b, c, d};
        } else {
            alignas(8) uint16_t h[4];
#pragma unroll
            for (int i = 0; i < 4; i++) h[i] = DT == PT_BFLOAT16 ? float_to_bf16(v[i]) : float_to_f16(v[i]);
            *(uint64_t *)p = *(const uint64_t *)h;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (e + i < size) store_c<DT>(p, (size_t)i, v[i]);
}

// LDS bytes of two tiles in `bufs` buffers, and how many buffers fit.
constexpr int attn_tile_bytes(int rows, int dp, int es) { return rows * dp * es; }
constexpr int kAttnLds = 131072;

// ------------------------------------------------------------- forward
// Rows of a key head are its queries times its `group` query heads, row r =
// query r / group, head r % group, so that the heads that share keys share
// the staged tiles, and a single token's heads fill a block together.
//
// RW = 4: four waves of 32 rows each read every staged key.  RW = 1, for 32
// rows or fewer: the waves take a quarter of each tile's keys each, with a
// softmax of their own, and join their results at the end.
template <int DT, int DP, int RW> struct AttnFwdShape {
    static constexpr int ES = AttnT<DT>::ES, KW = 4 / RW;
    static constexpr int BN = RW == 1 ? 128 : (ES == 4 || DP == 256 ? 32 : 64);
    static constexpr int TILE = attn_tile_bytes(BN, DP, ES);
    static constexpr int NBUF = 4 * TILE <= kAttnLds ? 2 : 1;
    static constexpr bool kBuilt = 2 * NBUF * TILE <= kAttnLds;
    static constexpr int WGS = 2 * NBUF * TILE <= 65536 && DP <= 128 ? 2 : 1;
};

template <int DT, int DP, int RW, bool VEC>
__global__ __launch_bounds__(256, (AttnFwdShape<DT, DP, RW>::WGS)) void k_attention(AttnArgs g)
{
    using T = AttnT<DT>;
    using S = typename T::S;
    using Shape = AttnFwdShape<DT, DP, RW>;
    constexpr int BN = Shape::BN, NBUF = Shape::NBUF, KW = Shape::KW, NKB = BN / 32 / KW, BM = 32 * RW;
    constexpr int KS = DP * T::ES / 32, ND = DP / 32;
    __shared__ __attribute__((aligned(1024))) S k0[BN * DP];
    __shared__ __attribute__((aligned(1024))) S v0[BN * DP];
    __shared__ __attribute__((aligned(1024))) S k1[NBUF == 2 ? BN * DP : 8];
    __shared__ __attribute__((aligned(1024))) S v1[NBUF == 2 ? BN * DP : 8];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int rw = RW == 4 ? wave : 0, kw = RW == 4 ? 0 : wave;
    // the longest rows of a causal prompt first, its key heads side by side:
    // where their number is a multiple of 8 each keeps to one XCD's L2
    const int nh = g.batch * g.kv_heads, tiles = (int)(gridDim.x / (unsigned)nh);
    const int tile = tiles - 1 - (int)blockIdx.x / nh, bh = (int)blockIdx.x % nh, b = bh / g.kv_heads, hk = bh % g.kv_heads;
    const int split = blockIdx.y;
    const AttnSeq sq = attn_seq(g.q_starts, g.q_lengths, g.q_rows, g.nq, b);
    const AttnSeq sk = attn_seq(g.k_starts, g.k_lengths, g.k_rows, g.nk, b);
    const int rows = sq.n * g.group, row0 = tile * BM;
    if (row0 >= rows) return;  // whole workgroup
    const int row = row0 + rw * 32 + (lane & 31), qi = row / g.group, hq = hk * g.group + row % g.group;
    const bool live = row < rows;

    typename T::Frag q[KS];
    attn_row<DT, DP, VEC>(q, (const S *)g.q + b * g.q_bs + (sq.row + qi) * g.q_ts + hq * g.q_hs, live, g.size, half);

    const AttnSrc ks = {(const char *)((const S *)g.k + b * g.k_bs + sk.row * g.k_ts + hk * g.k_hs), g.k_ts * T::ES, sk.n};
    const AttnSrc vs = {(const char *)((const S *)g.v + b * g.v_bs + sk.row * g.v_ts + hk * g.v_hs), g.v_ts * T::ES, sk.n};
    AttnStage<DT, DP, BN, 4, VEC> kl, vl;
    kl.init(ks, g.size, wave, lane);
    vl.init(vs, g.size, wave, lane);

    // keys that this row, the tile's first row and its last row see
    const int shift = sk.n - sq.n + 1;
    const int lim = g.causal ? min(sk.n, qi + shift) : sk.n;
    const int lim_first = g.causal ? min(sk.n, row0 / g.group + shift) : sk.n;
    const int lim_last = g.causal ? min(sk.n, (min(row0 + BM, rows) - 1) / g.group + shift) : sk.n;
    int t0 = 0, t1 = max(0, (lim_last + BN - 1) / BN);
    if (g.splits > 1) {
        const int most = (sk.n + BN - 1) / BN, per = (most + g.splits - 1) / g.splits;
        t0 = split * per;
        t1 = min(t1, t0 + per);
    }

    float m = -INFINITY, l = 0.0f;
    floatx16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] = 0.0f;

    AttnLane<DT, DP> at;
    at.init(lane);
    auto step = [&](int t, const S *kt, const S *vt) {
        at.fresh();
        floatx16 s[NKB];
#pragma unroll
        for (int kb = 0; kb < NKB; kb++) s[kb] = attn_rows<DT, DP>(kt, (kw * NKB + kb) * 32, q, at);
        const int key0 = t * BN + kw * NKB * 32 + 4 * half;
        if ((t + 1) * BN > lim_first) {  // uniform: some row does not see some key
#pragma unroll
            for (int kb = 0; kb < NKB; kb++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    s[kb][r] = key0 + kb * 32 + 8 * (r / 4) + r % 4 < lim ? s[kb][r] : -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int kb = 0; kb < NKB; kb++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[kb][r]);
        top = fmaxf(top, attn_other(top, lane)) * g.scale_log2;
        // The reference m of the exponentials follows the maximum only when
        // it is passed by more than 8 (a factor of 256): sums and products
        // are fp32 and a probability keeps its relative precision whatever
        // its size, so most tiles need no rescaling of the sums.
        if (!__all(!(top > m + 8.0f))) {
            const float to = fmaxf(m, top), a = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= a;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[d][e] *= a;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int kb = 0; kb < NKB; kb++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[kb][r] = __builtin_amdgcn_exp2f(fmaf(s[kb][r], g.scale_log2, -ref));
                l += s[kb][r];
            }
#pragma unroll
        for (int kb = 0; kb < NKB; kb++) attn_cols<DT, DP>(o, vt, (kw * NKB + kb) * 32, s[kb], at);
    };
    auto load = [&](int t, S *kt, S *vt) {
        kl.load(ks, g.size, t * BN, kt, wave, lane);
        vl.load(vs, g.size, t * BN, vt, wave, lane);
    };
    if constexpr (NBUF == 2) {
        if (t0 < t1) load(t0, k0, v0);
        for (int t = t0; t < t1; t += 2) {
            attn_landed();  // tile t has landed, and every wave is done with the other buffer
            if (t + 1 < t1) load(t + 1, k1, v1);
            step(t, k0, v0);
            if (t + 1 >= t1) break;
            attn_landed();
            if (t + 2 < t1) load(t + 2, k0, v0);
            step(t + 1, k1, v1);
        }
    } else {
        for (int t = t0; t < t1; t++) {
            attn_landed();
            load(t, k0, v0);
            attn_landed();
            step(t, k0, v0);
        }
    }

    l += attn_other(l, lane);
    if constexpr (KW > 1) {
        // join the waves: rescale to the common maximum, add through LDS
        __shared__ float ml[2][KW][32];
        __syncthreads();
        if (lane < 32) {
            ml[0][kw][lane] = m;
            ml[1][kw][lane] = l;
        }
        __syncthreads();
        float to = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < KW; w++) to = fmaxf(to, ml[0][w][lane & 31]);
        const float ref = to == -INFINITY ? 0.0f : to;
#pragma unroll
        for (int w = 0; w < KW; w++) sum += ml[1][w][lane & 31] * __builtin_amdgcn_exp2f(ml[0][w][lane & 31] - ref);
        const float a = __builtin_amdgcn_exp2f(m - ref);
        m = to;
        l = sum;
        // [wave][element][row] in the first buffer, one wave at a time per 32 elements: KW * 32 * 32 floats fit it
        float *box = (float *)k0;
        static_assert(KW * 1024 * 4 <= BN * DP * T::ES, "the joined block fits a tile");
#pragma unroll
        for (int d = 0; d < ND; d++) {
            if (d) __syncthreads();
#pragma unroll
            for (int e = 0; e < 16; e++) box[kw * 1024 + e * 64 + lane] = o[d][e] * a;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 16; e++) {
                float x = 0.0f;
#pragma unroll
                for (int w = 0; w < KW; w++) x += box[w * 1024 + e * 64 + lane];
                o[d][e] = x;
            }
        }
        if (kw) return;  // wave 0 writes
    }
    if (!live) return;
    if (g.splits > 1) {
        const long long at = ((long long)split * nh + bh) * ((long long)g.nq * g.group) + row;
        if (half == 0) *(attn_f32x2 *)(g.part_ml + at * 2) = attn_f32x2{m, l};
        if (l != 0.0f || l != l)  // nothing seen: nothing is read there
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    attn_store4<PT_FLOAT32>(g.part_o + at * g.size, d * 32 + 8 * e + 4 * half, g.size, o[d][4 * e],
                                            o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]);
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    S *to = (S *)g.out + b * g.o_bs + (sq.row + qi) * g.o_ts + hq * g.o_hs;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            attn_store4<DT>(to, d * 32 + 8 * e + 4 * half, g.size, o[d][4 * e] * inv, o[d][4 * e + 1] * inv,
                            o[d][4 * e + 2] * inv, o[d][4 * e + 3] * inv);
    if (g.lse && half == 0) {
        const long long stat = (g.q_starts ? sq.row : (long long)b * g.heads * g.nq) + (long long)hq * g.stat_rows + qi;
        g.lse[stat] = l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
    }
}

// ------------------------------------------- gradient of keys and values
// A wave keeps 32 keys and their values and streams the queries that see
// them, head by head of the group, so the sum over heads that share a key
// stays in its registers and no order of additions can change.
//
// PASS 0 computes both gradients.  float32 heads past 128 elements, whose
// two rows and two sums together would pass the register file, take PASS 1
// (values) and PASS 2 (keys).
template <int DT, int DP> struct AttnBwdShape {
    static constexpr int ES = AttnT<DT>::ES;
    static constexpr int BQ = ES == 4 || DP == 256 ? 32 : 64;
    static constexpr int BN = BQ;
    static constexpr int TILE = attn_tile_bytes(BQ, DP, ES);
    static constexpr int WGS = 4 * TILE <= 65536 && DP * ES <= 128 ? 2 : 1;
    static constexpr bool kSplitPasses = DP * ES > 512;
};

// Four bytes a lane into LDS, zeros past `range`.
__device__ __forceinline__ void attn_load_lds4(const void *base, uint32_t off, float *lds, uint32_t range)
{
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)range, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (PT_LDS_AS void *)lds, 4, off, 0, 0, 0);
}

template <int DT, int DP, int PASS, bool VEC>
__global__ __launch_bounds__(256, (AttnBwdShape<DT, DP>::WGS)) void k_attention_dkv(AttnArgs g)
{
    using T = AttnT<DT>;
    using S = typename T::S;
    constexpr int BQ = AttnBwdShape<DT, DP>::BQ, NQB = BQ / 32, KS = DP * T::ES / 32, ND = DP / 32;
    constexpr bool kV = PASS != 2, kK = PASS != 1;
    __shared__ __attribute__((aligned(1024))) S q0[BQ * DP], w0[BQ * DP], q1[BQ * DP], w1[BQ * DP];
    __shared__ __attribute__((aligned(256))) float l0[64], l1[64], e0[64], e1[64];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    // the first keys of a causal sequence, which most queries see, first
    const int nh = g.batch * g.kv_heads;
    const int tile = (int)blockIdx.x / nh, bh = (int)blockIdx.x % nh, b = bh / g.kv_heads, hk = bh % g.kv_heads;
    const AttnSeq sq = attn_seq(g.q_starts, g.q_lengths, g.q_rows, g.nq, b);
    const AttnSeq sk = attn_seq(g.k_starts, g.k_lengths, g.k_rows, g.nk, b);
    const int first = tile * 128;
    if (first >= sk.n) return;  // whole workgroup
    const int key = first + wave * 32 + (lane & 31);
    const bool live = key < sk.n;
    typename T::Frag k[KS], v[kK ? KS : 1];
    attn_row<DT, DP, VEC>(k, (const S *)g.k + b * g.k_bs + (sk.row + key) * g.k_ts + hk * g.k_hs, live, g.size, half);
    if constexpr (kK)
        attn_row<DT, DP, VEC>(v, (const S *)g.v + b * g.v_bs + (sk.row + key) * g.v_ts + hk * g.v_hs, live, g.size, half);

    // query i sees key j where i >= j - shift
    const int shift = sk.n - sq.n;
    const int from = g.causal ? key - shift : INT_MIN;
    const int t0 = g.causal ? max(0, first - shift) / BQ : 0, per = max(0, (sq.n + BQ - 1) / BQ - t0);
    const int steps = per * g.group;

    floatx16 dk[kK ? ND : 1], dv[kV ? ND : 1];
#pragma unroll
    for (int e = 0; e < 16; e++) {
#pragma unroll
        for (int d = 0; d < (kK ? ND : 1); d++) dk[d][e] = 0.0f;
#pragma unroll
        for (int d = 0; d < (kV ? ND : 1); d++) dv[d][e] = 0.0f;
    }

    const S *qb = (const S *)g.q + b * g.q_bs + sq.row * g.q_ts, *wb = (const S *)g.w + b * g.o_bs + sq.row * g.o_ts;
    const long long stat = g.q_starts ? sq.row : (long long)b * g.heads * g.nq;
    AttnStage<DT, DP, BQ, 4, VEC> ql, wl;
    ql.init({nullptr, g.q_ts * T::ES, 0}, g.size, wave, lane);
    wl.init({nullptr, g.o_ts * T::ES, 0}, g.size, wave, lane);
    auto load = [&](int it, S *qt, S *wt, float *lt, float *et) {
        const int hq = hk * g.group + it / per, r0 = (t0 + it % per) * BQ;
        ql.load({(const char *)(qb + hq * g.q_hs), g.q_ts * T::ES, sq.n}, g.size, r0, qt, wave, lane);
        wl.load({(const char *)(wb + hq * g.o_hs), g.o_ts * T::ES, sq.n}, g.size, r0, wt, wave, lane);
        const long long at = stat + (long long)hq * g.stat_rows + r0;
        const uint32_t range = (uint32_t)min(sq.n - r0, BQ) * 4u;
        // rows past the last have zero products; a zero lse keeps their exponentials finite
        if (wave == 0) attn_load_lds4(g.lse2 + at, lane * 4u, lt, range);
        if (wave == 1) attn_load_lds4(g.delta + at, lane * 4u, et, range);
    };
    AttnLane<DT, DP> at;
    at.init(lane);
    auto step = [&](int it, const S *qt, const S *wt, const float *lt, const float *et) {
        at.fresh();
        const int i0 = (t0 + it % per) * BQ + 4 * half;
        const bool mask = g.causal && (t0 + it % per) * BQ < first + 127 - shift;
#pragma unroll
        for (int qb2 = 0; qb2 < NQB; qb2++) {
            floatx16 p = attn_rows<DT, DP>(qt, qb2 * 32, k, at);
#pragma unroll
            for (int r4 = 0; r4 < 4; r4++) {
                const floatx4 ls = *(const floatx4 *)(lt + qb2 * 32 + 8 * r4 + 4 * half);
#pragma unroll
                for (int x = 0; x < 4; x++)
                    p[4 * r4 + x] = __builtin_amdgcn_exp2f(fmaf(p[4 * r4 + x], g.scale_log2, -ls[x]));
            }
            if (mask) {
#pragma unroll
                for (int r = 0; r < 16; r++) p[r] = i0 + qb2 * 32 + 8 * (r / 4) + r % 4 >= from ? p[r] : 0.0f;
            }
            if constexpr (kV) attn_cols<DT, DP>(dv, wt, qb2 * 32, p, at);
            if constexpr (kK) {
                floatx16 t = attn_rows<DT, DP>(wt, qb2 * 32, v, at);
#pragma unroll
                for (int r4 = 0; r4 < 4; r4++) {
                    const floatx4 es = *(const floatx4 *)(et + qb2 * 32 + 8 * r4 + 4 * half);
#pragma unroll
                    for (int x = 0; x < 4; x++) t[4 * r4 + x] = p[4 * r4 + x] * (t[4 * r4 + x] - es[x]);
                }
                attn_cols<DT, DP>(dk, qt, qb2 * 32, t, at);
            }
        }
    };
    if (steps) load(0, q0, w0, l0, e0);
    for (int it = 0; it < steps; it += 2) {
        attn_landed();  // this step's tiles are there, and every wave is done with the other buffer
        if (it + 1 < steps) load(it + 1, q1, w1, l1, e1);
        step(it, q0, w0, l0, e0);
        if (it + 1 >= steps) break;
        attn_landed();
        if (it + 2 < steps) load(it + 2, q0, w0, l0, e0);
        step(it + 1, q1, w1, l1, e1);
    }
    if (!live) return;
    // gradients are contiguous
    const long long to = ((g.k_starts ? sk.row + key : (long long)b * g.nk + key) * g.kv_heads + hk) * g.size;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (kV)
                attn_store4<DT>((S *)g.dv + to, d * 32 + 8 * e + 4 * half, g.size, dv[d][4 * e], dv[d][4 * e + 1],
                                dv[d][4 * e + 2], dv[d][4 * e + 3]);
            if constexpr (kK)
                attn_store4<DT>((S *)g.dk + to, d * 32 + 8 * e + 4 * half, g.size, dk[d][4 * e] * g.scale,
                                dk[d][4 * e + 1] * g.scale, dk[d][4 * e + 2] * g.scale, dk[d][4 * e + 3] * g.scale);
        }
}

// ------------------------------------------------- gradient of the queries
// Rows as in the forward pass; the keys and values stream past them.
template <int DT, int DP, bool VEC>
__global__ __launch_bounds__(256, (AttnBwdShape<DT, DP>::WGS)) void k_attention_dq(AttnArgs g)
{
    using T = AttnT<DT>;
    using S = typename T::S;
    constexpr int BN = AttnBwdShape<DT, DP>::BN, NKB = BN / 32, KS = DP * T::ES / 32, ND = DP / 32, BM = 128;
    __shared__ __attribute__((aligned(1024))) S k0[BN * DP], v0[BN * DP], k1[BN * DP], v1[BN * DP];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int nh = g.batch * g.kv_heads, tiles = (int)(gridDim.x / (unsigned)nh);
    const int tile = tiles - 1 - (int)blockIdx.x / nh, bh = (int)blockIdx.x % nh, b = bh / g.kv_heads, hk = bh % g.kv_heads;
    const AttnSeq sq = attn_seq(g.q_starts, g.q_lengths, g.q_rows, g.nq, b);
    const AttnSeq sk = attn_seq(g.k_starts, g.k_lengths, g.k_rows, g.nk, b);
    const int rows = sq.n * g.group, row0 = tile * BM;
    if (row0 >= rows) return;  // whole workgroup
    const int row = row0 + wave * 32 + (lane & 31), qi = row / g.group, hq = hk * g.group + row % g.group;
    const bool live = row < rows;

    typename T::Frag q[KS], w[KS];
    attn_row<DT, DP, VEC>(q, (const S *)g.q + b * g.q_bs + (sq.row + qi) * g.q_ts + hq * g.q_hs, live, g.size, half);
    attn_row<DT, DP, VEC>(w, (const S *)g.w + b * g.o_bs + (sq.row + qi) * g.o_ts + hq * g.o_hs, live, g.size, half);
    const long long stat = (g.q_starts ? sq.row : (long long)b * g.heads * g.nq) + (long long)hq * g.stat_rows + qi;
    const float ls = live ? g.lse2[stat] : INFINITY, es = live ? g.delta[stat] : 0.0f;

    const AttnSrc ks = {(const char *)((const S *)g.k + b * g.k_bs + sk.row * g.k_ts + hk * g.k_hs), g.k_ts * T::ES, sk.n};
    const AttnSrc vs = {(const char *)((const S *)g.v + b * g.v_bs + sk.row * g.v_ts + hk * g.v_hs), g.v_ts * T::ES, sk.n};
    AttnStage<DT, DP, BN, 4, VEC> kl, vl;
    kl.init(ks, g.size, wave, lane);
    vl.init(vs, g.size, wave, lane);
    const int shift = sk.n - sq.n + 1;
    const int lim = g.causal ? min(sk.n, qi + shift) : sk.n;
    const int lim_first = g.causal ? min(sk.n, row0 / g.group + shift) : sk.n;
    const int lim_last = g.causal ? min(sk.n, (min(row0 + BM, rows) - 1) / g.group + shift) : sk.n;
    const int t1 = max(0, (lim_last + BN - 1) / BN);

    floatx16 dq[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) dq[d][e] = 0.0f;
    AttnLane<DT, DP> at;
    at.init(lane);
    auto step = [&](int t, const S *kt, const S *vt) {
        at.fresh();
        const int key0 = t * BN + 4 * half;
        const bool mask = (t + 1) * BN > lim_first;
#pragma unroll
        for (int kb = 0; kb < NKB; kb++) {
            floatx16 p = attn_rows<DT, DP>(kt, kb * 32, q, at);
#pragma unroll
            for (int r = 0; r < 16; r++) p[r] = __builtin_amdgcn_exp2f(fmaf(p[r], g.scale_log2, -ls));
            if (mask) {
#pragma unroll
                for (int r = 0; r < 16; r++) p[r] = key0 + kb * 32 + 8 * (r / 4) + r % 4 < lim ? p[r] : 0.0f;
            }
            floatx16 x = attn_rows<DT, DP>(vt, kb * 32, w, at);
#pragma unroll
            for (int r = 0; r < 16; r++) x[r] = p[r] * (x[r] - es);
            attn_cols<DT, DP>(dq, kt, kb * 32, x, at);
        }
    };
    auto load = [&](int t, S *kt, S *vt) {
        kl.load(ks, g.size, t * BN, kt, wave, lane);
        vl.load(vs, g.size, t * BN, vt, wave, lane);
    };
    if (t1 > 0) load(0, k0, v0);
    for (int t = 0; t < t1; t += 2) {
        attn_landed();  // tile t has landed, and every wave is done with the other buffer
        if (t + 1 < t1) load(t + 1, k1, v1);
        step(t, k0, v0);
        if (t + 1 >= t1) break;
        attn_landed();
        if (t + 2 < t1) load(t + 2, k0, v0);
        step(t + 1, k1, v1);
    }
    if (!live) return;
    S *to = (S *)g.dq + b * g.o_bs + (sq.row + qi) * g.o_ts + hq * g.o_hs;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            attn_store4<DT>(to, d * 32 + 8 * e + 4 * half, g.size, dq[d][4 * e] * g.scale, dq[d][4 * e + 1] * g.scale,
                            dq[d][4 * e + 2] * g.scale, dq[d][4 * e + 3] * g.scale);
}

// ------------------------------------------------------------- launches
// Of one element type (pt_attention_{bf16,f16,f32}.hip).  `vec`: every row
// of every operand starts on 16 bytes and its size fills whole chunks.
template <int DT> void launch_attention(const AttnArgs &g, bool narrow, bool vec, unsigned blocks, hipStream_t s);
template <int DT> void launch_attention_dkv(const AttnArgs &g, bool vec, unsigned blocks, hipStream_t s);
template <int DT> void launch_attention_dq(const AttnArgs &g, bool vec, unsigned blocks, hipStream_t s);
// whether 32 rows or fewer have a kernel of their own (RW = 1) at this size
template <int DT> bool attention_narrow_built(int size);

}  // namespace pt
