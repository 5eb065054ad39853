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
#include <type_traits>

#include "pt_gemm.h"

namespace pt {

struct AttnArgs {
    const void *q, *k, *v;
    void *out, *rest;
    float *lse;
    // strides in elements: sequence (0 where starts are given), token, head
    long long q_bs, q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs, o_bs, o_ts, o_hs;
    const int32_t *q_starts, *q_lengths, *k_starts, *k_lengths;  // device, or null
    int batch, heads, kv_heads, group, size, nq, nk, q_rows, k_rows;
    int causal;
    float scale, scale_log2;
    int splits;               // key ranges computed by workgroups of their own
    // their results: [split][part_step rows][size], and (m, l), as attn_far_part says; a row is one of a sequence and
    // key head, or (part_packed) a token row's head
    float *part_o, *part_ml;
    int part_packed;
    int place, tiles;         // AttnPlace, and the tiles of a head
    long long part_step;      // backward: parts of dk or dq in part_o, of dv in part_ml, this many elements apart
    // backward
    const void *w;            // upstream gradient in the element type, contiguous like out
    // per (head, token row): lse in base 2 (+inf where nothing is seen), d, and what scores lose first (kExactLse)
    float *lse2, *delta, *tops;
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

// Which tile, sequence and key head a workgroup takes, the longest work
// first.  Workgroups go to the 8 XCDs in turn; each XCD has an L2 of 4 MB,
// which holds the keys and values of a head or two.
enum AttnPlace {
    // the tiles of all heads side by side
    kPlain = 0,
    // Heads a multiple of 8: a head keeps to an XCD, which takes as many heads
    // at once as fill its 64 workgroups and the next when those run out.  A
    // causal head's tiles fall in length, so the next heads' long ones follow
    // the last's short ones.
    kGrouped,
    // Key heads a divisor of 8: the XCDs divide the key heads between them,
    // and those with one head its tiles, so every sequence loads all of them.
    kSpread,
    // Sequences of different lengths: the tiles that exist, numbered through
    // all sequences by their distance from the short end, the key heads to
    // the XCDs as above.  Numbering tiles that do not exist too leaves
    // workgroups empty, which come at a period of the dispatch and leave
    // whole shader engines idle (225 us instead of 153 for six prompts of
    // 4096 to 1 tokens).
    kRagged
};

// The item-th of the existing tiles, from the highest level down: level t
// holds the t-th tile of every sequence that has one.  The tiles at level t
// and above number sum over sequences of max(0, tiles - t).
__device__ __forceinline__ bool attn_item(const int32_t *starts, const int32_t *lengths, int rows, int most, int batch,
                                          int group, int levels, int item, int &level, int &b)
{
    const int lane = threadIdx.x & 63;
    auto tiles = [&](int i) { return i < batch ? (int)(((long long)attn_seq(starts, lengths, rows, most, i).n * group + 127) / 128) : 0; };
    const int first = tiles(lane);
    auto above = [&](int t) {
        int n = max(0, first - t);
        for (int i = lane + 64; i < batch; i += 64) n += max(0, tiles(i) - t);
        return wave_all(n, FAdd{});
    };
    if (item >= above(0)) return false;
    int low = 0, high = levels;
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (above(mid) > item) low = mid;
        else high = mid;
    }
    int r = item - above(low + 1);
    for (int c = 0; c < batch; c += 64) {
        const bool has = (c ? tiles(c + lane) : first) > low;
        const uint64_t mask = __ballot(has);
        const int n = (int)__popcll(mask);
        if (r < n) {
            const uint64_t it = __ballot(has && (int)__popcll(mask & ((1ull << lane) - 1)) == r);
            level = low;
            b = c + (int)__builtin_ctzll(it);
            return true;
        }
        r -= n;
    }
    return false;
}

// `keys`: tiles of the keys, whose first is the longest work (the queries'
// last is).  false: nothing for this workgroup.
__device__ __forceinline__ bool attn_place(const AttnArgs &g, bool keys, int &tile, int &bh)
{
    const unsigned id = blockIdx.x, nh = (unsigned)(g.batch * g.kv_heads), tiles = (unsigned)g.tiles, kv = (unsigned)g.kv_heads;
    const unsigned x = id % 8, j = id / 8;
    if (g.place == kRagged) {
        unsigned item = id / kv, h = id % kv;
        if (8 % kv == 0) {
            item = j * (8 / kv) + x % (8 / kv);
            h = x / (8 / kv);
        } else if (kv % 8 == 0) {
            item = j / (kv / 8);
            h = x + j % (kv / 8) * 8;
        }
        int t, b;
        const bool some = keys ? attn_item(g.k_starts, g.k_lengths, g.k_rows, g.nk, g.batch, 1, g.tiles, (int)item, t, b)
                               : attn_item(g.q_starts, g.q_lengths, g.q_rows, g.nq, g.batch, g.group, g.tiles, (int)item, t, b);
        if (!some) return false;
        t = __builtin_amdgcn_readfirstlane(t);
        b = __builtin_amdgcn_readfirstlane(b);
        if (keys) t = (attn_seq(g.k_starts, g.k_lengths, g.k_rows, g.nk, b).n + 127) / 128 - 1 - t;
        tile = t;
        bh = b * g.kv_heads + (int)h;
        return true;
    }
    unsigned t = id / nh, h = id % nh;
    if (g.place == kGrouped) {
        const unsigned heads = nh / 8, most = min(heads, max(1u, 64 / tiles));
        const unsigned first = j / (tiles * most) * most, n = min(most, heads - first), r = j - first * tiles;
        t = r / n;
        h = (first + r % n) * 8 + x;
    } else if (g.place == kSpread) {
        t = j / (unsigned)g.batch * (8 / kv) + x % (8 / kv);
        h = j % (unsigned)g.batch * kv + x / (8 / kv);
    }
    if (t >= tiles) return false;
    tile = (int)(keys ? t : tiles - 1 - t);
    bh = (int)h;
    return true;
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
    // bytes from row r0 on that hold rows of the source, for loads of whole
    // tiles no bound: the compiler's 64-bit product is kept for the last tile
    __device__ __forceinline__ static uint32_t range(const AttnSrc &s, int size, int r0)
    {
        uint32_t bytes = 0x7fffffffu;
        if (__builtin_expect(r0 + ROWS > s.rows, 0))
            bytes = r0 >= s.rows ? 0u : (uint32_t)(s.rows - r0 - 1) * (uint32_t)s.step + (uint32_t)(size * T::ES);
        return bytes;
    }
    // The same chunks to registers; read once.
    __device__ __forceinline__ void fetch(const AttnSrc &s, int size, int r0, floatx4 (&v)[NI]) const
    {
        static_assert(VEC, "whole packs");
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char *>(s.base + (unsigned long long)(uint32_t)r0 * (uint32_t)s.step), (short)0, (int)range(s, size, r0), 0x00020000);
#pragma unroll
        for (int i = 0; i < NI; i++)
            v[i] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off[i], 0, 2));  // nt
    }
    // Rows r0 .. r0 + ROWS - 1 into `tile`; rows past the source's last are zeros.
    __device__ __forceinline__ void load(const AttnSrc &s, int size, int r0, S *tile, int wave, int lane) const
    {
        // (a step fits 32 bits where rows come in whole packs)
        const char *base = s.base + (VEC ? (unsigned long long)(uint32_t)r0 * (uint32_t)s.step : (unsigned long long)r0 * s.step);
        if constexpr (VEC) {
            const uint32_t bytes = range(s, size, r0);
#pragma unroll
            for (int i = 0; i < NI; i++)
                buffer_load_lds16(base, off[i], (PT_LDS_AS void *)(tile + (wave * NI + i) * 64 * T::PK), bytes);
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

// The other half's value of the same column.
__device__ __forceinline__ float attn_other(float v, int lane)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(lane < 32 ? r[1] : r[0]);
}

// acc + a . b
template <int DT>
__device__ __forceinline__ float attn_dot(const typename AttnT<DT>::Frag &a, const typename AttnT<DT>::Frag &b, float acc)
{
    using S = typename AttnT<DT>::S;
    struct E { S s[AttnT<DT>::PK]; };
    const E x = __builtin_bit_cast(E, a), y = __builtin_bit_cast(E, b);
#pragma unroll
    for (int e = 0; e < AttnT<DT>::PK; e++) acc = fmaf(DType<DT>::to_c(x.s[e]), DType<DT>::to_c(y.s[e]), acc);
    return acc;
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

// Chunk 2 t + lane / 32 of tile row row0 + lane % 32: the left operand's
// fragment t of the product over the head's size.
template <int DT, int DP>
__device__ __forceinline__ typename AttnT<DT>::Frag attn_row_frag(const typename AttnT<DT>::S *tile, int row0, int t,
                                                                  const AttnLane<DT, DP> &at)
{
    const PT_LDS_AS char *base = (const PT_LDS_AS char *)tile + row0 * DP * AttnT<DT>::ES;
    return __builtin_bit_cast(typename AttnT<DT>::Frag, *(const PT_LDS_AS floatx4 *)(base + (at.row ^ (uint32_t)(t << 5))));
}

// acc[streamed row][own row] = sum over the head's size, for the 32 tile
// rows from row0.
template <int DT, int DP>
__device__ __forceinline__ floatx16 attn_rows(const typename AttnT<DT>::S *tile, int row0,
                                              const typename AttnT<DT>::Frag (&b)[DP * AttnT<DT>::ES / 32],
                                              const AttnLane<DT, DP> &at)
{
    floatx16 acc;
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] = 0.0f;
#pragma unroll
    for (int t = 0; t < DP * AttnT<DT>::ES / 32; t++) attn_mfma<DT>(acc, attn_row_frag<DT, DP>(tile, row0, t, at), b[t]);
    return acc;
}

typedef float attn_f32x2 __attribute__((ext_vector_type(2)));
typedef float attn_f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 attn_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 attn_f16x8 __attribute__((ext_vector_type(8)));

// Registers 8 u .. 8 u + 7 of a block rounded to the element type: the right
// operand of the product over the streamed rows.  The products take 16-bit
// operands, and one rounding here costs about what the result's own does
// (together 1.4 times the error).  In float16 gradients of scores below 2^-14
// lose bits and below 2^-25 vanish, as gradients of that size do themselves.
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
//
// Unit u of 2 * DP / 32 (16-bit: rows 16 (u / blocks) .. + 15, element block
// u % blocks) or of 16 * DP / 32 (float32: register u / blocks).
template <int DT, int DP> constexpr int attn_col_units() { return (DT == PT_FLOAT32 ? 16 : 2) * DP / 32; }
template <int DT> using AttnColFrag = std::conditional_t<DT == PT_FLOAT32, float, typename AttnT<DT>::Frag>;

template <int DT, int DP>
__device__ __forceinline__ AttnColFrag<DT> attn_col_frag(const typename AttnT<DT>::S *tile, int row0, int u,
                                                         const AttnLane<DT, DP> &at)
{
    using T = AttnT<DT>;
    const PT_LDS_AS char *base = (const PT_LDS_AS char *)tile + row0 * DP * T::ES;
    const int d = u % (DP / 32), r = u / (DP / 32);
    if constexpr (DT == PT_FLOAT32) {
        // row 8 (r / 4) + r % 4 (+ 4 half): the swizzle's bits of r, the half's are in the base
        const int x = (r % 4) << 2 | ((r / 4) * 2 & 3);
        return *(const PT_LDS_AS float *)(base + (8 * (r / 4) + r % 4) * DP * 4 + (at.col0 ^ (uint32_t)((8 * d ^ x) << 4)));
    } else {
        typedef short v4s __attribute__((ext_vector_type(4)));
        const PT_LDS_AS char *to = base + r * 16 * DP * T::ES;
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((PT_LDS_AS v4s *)(to + (at.col0 ^ (uint32_t)(d << 6))));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((PT_LDS_AS v4s *)(to + (at.col1 ^ (uint32_t)(d << 6))));
        return __builtin_bit_cast(typename T::Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

// The right operand of unit u's rows.
template <int DT, int DP>
__device__ __forceinline__ AttnColFrag<DT> attn_col_right(const floatx16 &p, int u)
{
    if constexpr (DT == PT_FLOAT32) return p[u / (DP / 32)];
    else return attn_pack<DT>(p, u / (DP / 32));
}

template <int DT, int DP>
__device__ __forceinline__ void attn_col_mfma(floatx16 (&acc)[DP / 32], int u, const AttnColFrag<DT> &a, const AttnColFrag<DT> &b)
{
    floatx16 &x = acc[u % (DP / 32)];
    if constexpr (DT == PT_FLOAT32) x = __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, x, 0, 0, 0);
    else attn_mfma<DT>(x, a, b);
}

template <int DT, int DP>
__device__ __forceinline__ void attn_cols(floatx16 (&acc)[DP / 32], const typename AttnT<DT>::S *tile, int row0,
                                          const floatx16 &p, const AttnLane<DT, DP> &at)
{
#pragma unroll
    for (int u = 0; u < attn_col_units<DT, DP>(); u++)
        attn_col_mfma<DT, DP>(acc, u, attn_col_frag<DT, DP>(tile, row0, u, at), attn_col_right<DT, DP>(p, u));
}

// A fragment of either product, for a queue that reads ahead across both.
template <int DT>
__device__ __forceinline__ typename AttnT<DT>::Frag attn_any(const AttnColFrag<DT> &a)
{
    if constexpr (DT == PT_FLOAT32) return floatx4{a, 0.0f, 0.0f, 0.0f};
    else return a;
}
template <int DT>
__device__ __forceinline__ AttnColFrag<DT> attn_of_any(const typename AttnT<DT>::Frag &a)
{
    if constexpr (DT == PT_FLOAT32) return a[0];
    else return a;
}

// Units 0 .. N - 1 of MFMA work in this order, fragment(unit) read AHEAD units
// before unit(unit, fragment) uses it; unit() also does what other work runs
// beside the matrix pipe.  Nothing moves from unit to unit: the order bounds
// the fragments that are held, and left to itself the compiler reads so far
// ahead that registers spill, and sinks the work to where it is used.
template <int DT, int N, int AHEAD, typename F, typename U>
__device__ __forceinline__ void attn_queue(F &&fragment, U &&unit)
{
    typename AttnT<DT>::Frag f[AHEAD + 1];
    static_for<0, AHEAD>([&](auto I) __attribute__((always_inline)) { f[decltype(I)::value] = fragment(I); });
    __builtin_amdgcn_sched_barrier(0);
    static_for<0, N>([&](auto I) __attribute__((always_inline)) {
        constexpr int u = decltype(I)::value, w = u + AHEAD;
        if constexpr (w < N) f[w % (AHEAD + 1)] = fragment(IC<w>{});
        unit(I, f[u % (AHEAD + 1)]);
        __builtin_amdgcn_sched_barrier(0);
    });
}

// The same products with other work beside them: after each unit's MFMA,
// work(unit) runs while the matrix pipe does, and nothing moves across.  The
// order also bounds the fragments that are held at once; left to itself the
// compiler reads so far ahead that the gradient kernels spill.
template <int DT, int DP, int AHEAD, typename B, typename W>
__device__ __forceinline__ void attn_rows_beside(floatx16 &acc, const typename AttnT<DT>::S *tile, int row0, B &&right,
                                                 const AttnLane<DT, DP> &at, W &&work)
{
    constexpr int N = DP * AttnT<DT>::ES / 32;
    typename AttnT<DT>::Frag a[AHEAD + 1], b[AHEAD + 1];
    static_for<0, AHEAD>([&](auto U) {
        constexpr int u = decltype(U)::value;
        a[u] = attn_row_frag<DT, DP>(tile, row0, u, at);
        b[u] = right(u);
    });
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] = 0.0f;
    static_for<0, N>([&](auto U) {
        constexpr int u = decltype(U)::value, w = u + AHEAD;
        if constexpr (w < N) {
            a[w % (AHEAD + 1)] = attn_row_frag<DT, DP>(tile, row0, w, at);
            b[w % (AHEAD + 1)] = right(w);
        }
        attn_mfma<DT>(acc, a[u % (AHEAD + 1)], b[u % (AHEAD + 1)]);
        work(U, IC<N>{});
        __builtin_amdgcn_sched_barrier(0);
    });
}

template <int DT, int DP, int AHEAD, typename W>
__device__ __forceinline__ void attn_cols_beside(floatx16 (&acc)[DP / 32], const typename AttnT<DT>::S *tile, int row0,
                                                 const floatx16 &p, const AttnLane<DT, DP> &at, W &&work)
{
    constexpr int N = attn_col_units<DT, DP>(), ND = DP / 32;
    AttnColFrag<DT> a[AHEAD + 1], b[N / ND];
#pragma unroll
    for (int u = 0; u < N; u += ND) b[u / ND] = attn_col_right<DT, DP>(p, u);
    static_for<0, AHEAD>([&](auto U) { a[decltype(U)::value] = attn_col_frag<DT, DP>(tile, row0, decltype(U)::value, at); });
    static_for<0, N>([&](auto U) {
        constexpr int u = decltype(U)::value, w = u + AHEAD;
        if constexpr (w < N) a[w % (AHEAD + 1)] = attn_col_frag<DT, DP>(tile, row0, w, at);
        attn_col_mfma<DT, DP>(acc, u, a[u % (AHEAD + 1)], b[u / ND]);
        work(U, IC<N>{});
        __builtin_amdgcn_sched_barrier(0);
    });
}

// Unit u of n does its share of 16 registers: f(register).
template <typename U, typename N, typename F>
__device__ __forceinline__ void attn_share(U, N, F &&f)
{
    static_for<U::value * 16 / N::value, (U::value + 1) * 16 / N::value>([&](auto E) { f(decltype(E)::value); });
}

// Everything this wave loads or writes to LDS is there, and every wave has
// come here: the loads to LDS are waited for by hand, since the compiler's
// own barrier need not wait for them.
__device__ __forceinline__ void attn_landed()
{
    ring_wait<0>();
    ring_barrier();
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

// A block's column in its contiguous row: register r holds element first +
// 8 (r / 4) + 4 half + r % 4, value(r) of it.  16 bits: the two lanes of a
// column change pieces so that each stores whole packs, half the stores and
// twice the bytes a row in each (all lanes that share a row come here).
template <int DT, typename F>
__device__ __forceinline__ void attn_store_block(void *row, int first, int size, int half, F &&value)
{
    if constexpr (DT != PT_FLOAT32) {
        typedef unsigned int u32x4 __attribute__((ext_vector_type(4), aligned(2)));
        if ((size & 7) == 0) {
            auto two = [&](int r) {
                const float x = value(r), y = value(r + 1);
                return DT == PT_BFLOAT16 ? (uint32_t)float_to_bf16(x) | (uint32_t)float_to_bf16(y) << 16
                                         : (uint32_t)float_to_f16(x) | (uint32_t)float_to_f16(y) << 16;
            };
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const auto a = __builtin_amdgcn_permlane32_swap(two(4 * e), two(4 * e + 4), false, false);
                const auto b = __builtin_amdgcn_permlane32_swap(two(4 * e + 2), two(4 * e + 6), false, false);
                const int at = first + 8 * (e + half);
                if (at < size) *(u32x4 *)((typename AttnT<DT>::S *)row + at) = u32x4{a[0], b[0], a[1], b[1]};
            }
            return;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        attn_store4<DT>(row, first + 8 * e + 4 * half, size, value(4 * e), value(4 * e + 1), value(4 * e + 2), value(4 * e + 3));
}

// What a rounding to the element type takes from x.
template <int DT> __device__ __forceinline__ float attn_rest(float x)
{
    return x - (DT == PT_BFLOAT16 ? bf16_to_float(float_to_bf16(x)) : f16_to_float(float_to_f16(x)));
}

// The reference of a row's exponentials is m = round(c s_max), c = scale
// log2(e), and the exponent fma(c, s, -m).  It is off by the rounding of m in
// every element of the row alike: a factor that the sum cancels, 2^0.5 at most
// while |m| <= 2^24.  Beyond, the factor itself would leave float16, and from
// 2^32 on float32 (float16 operands of some thousands give scores of 1e9).
// Rows with such a reference are far: their workgroup computes its rows once
// more by (s - s_max) c, in a plain loop behind the fast one.
constexpr float kFarScore = 16777216.0f;
__device__ __forceinline__ bool attn_far(float m) { return fabsf(m) > kFarScore && m != -INFINITY; }

// Is x (uniform in a wave) true in any of the W waves?  One barrier.
template <int W> __device__ __forceinline__ bool attn_any_wave(bool x, int lane, int wave)
{
    __shared__ int box[W];
    if (lane == 0) box[wave] = x;
    __syncthreads();
    int any = 0;
#pragma unroll
    for (int w = 0; w < W; w++) any |= box[w];
    return __builtin_amdgcn_readfirstlane(any) != 0;
}

// One block's scores (masked) into sums that are kept by (s - m) c, m the
// largest score so far.
template <int DT, int DP>
__device__ __forceinline__ void attn_far_block(floatx16 &s, float &m, float &l, floatx16 (&o)[DP / 32], float c,
                                               const typename AttnT<DT>::S *vt, int row0, const AttnLane<DT, DP> &at, int lane)
{
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; r++) top = fmaxf(top, s[r]);
    top = fmaxf(m, fmaxf(top, attn_other(top, lane)));
    const float ref = top == -INFINITY ? 0.0f : top, a = __builtin_amdgcn_exp2f((m - ref) * c);
    m = top;
    l *= a;
#pragma unroll
    for (int d = 0; d < DP / 32; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] *= a;
#pragma unroll
    for (int r = 0; r < 16; r++) {
        s[r] = __builtin_amdgcn_exp2f((s[r] - ref) * c);
        l += s[r];
    }
    attn_cols<DT, DP>(o, vt, row0, s, at);
}

// What these sums hand on.  m becomes round(c m) where that is the row's
// result.  A range's part of a far row keeps m as it is and says so by a
// negative l; of other rows it is as the fast loop leaves it.
template <int ND>
__device__ __forceinline__ void attn_far_part(float &m, float &l, floatx16 (&o)[ND], float c, bool part)
{
    const float mc = m * c;
    if (!part || m == -INFINITY) {
        m = mc;
    } else if (attn_far(mc)) {
        l = -l;
    } else {
        const float f = __builtin_amdgcn_exp2f(fmaf(m, c, -mc));
        m = mc;
        l *= f;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[d][e] *= f;
    }
}

// LDS bytes of a tile.
constexpr int attn_tile_bytes(int rows, int dp, int es) { return rows * dp * es; }

// Joins the waves' results in wave 0 and all others: rescaled to the common
// maximum, added through `box` (W * 1024 floats that nobody reads any more),
// 32 elements of the head at a time.  c: by what differences of m count.
template <int W, int ND>
__device__ __forceinline__ void attn_join_waves(float &m, float &l, floatx16 (&o)[ND], float c, float *box, int lane, int wave)
{
    __shared__ float ml[2][W][32];
    if (lane < 32) {
        ml[0][wave][lane] = m;
        ml[1][wave][lane] = l;
    }
    __syncthreads();
    float to = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) to = fmaxf(to, ml[0][w][lane & 31]);
    const float ref = to == -INFINITY ? 0.0f : to;
#pragma unroll
    for (int w = 0; w < W; w++) sum += ml[1][w][lane & 31] * __builtin_amdgcn_exp2f((ml[0][w][lane & 31] - ref) * c);
    const float a = __builtin_amdgcn_exp2f((m - ref) * c);
    m = to;
    l = sum;
#pragma unroll
    for (int d = 0; d < ND; d++) {
        if (d) __syncthreads();
#pragma unroll
        for (int e = 0; e < 16; e++) box[wave * 1024 + e * 64 + lane] = o[d][e] * a;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 16; e++) {
            float x = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) x += box[w * 1024 + e * 64 + lane];
            o[d][e] = x;
        }
    }
}

// The row among part_step that query qi of sequence b, query head hq has;
// row: the same among the sequence's and key head's.
__device__ __forceinline__ long long attn_part_row(const AttnArgs &g, int bh, int row, long long token, int hq)
{
    return g.part_packed ? token * g.heads + hq : bh * ((long long)g.nq * g.group) + row;
}

// A wave's rows: the output and lse, or one range's sums.
template <int DT, int ND>
__device__ __forceinline__ void attn_result(const AttnArgs &g, float m, float l, const floatx16 (&o)[ND], bool live, int b,
                                            int bh, int row, long long token, int qi, int hq, int split, int half)
{
    if (!live) return;
    if (g.splits > 1) {
        const long long at = split * g.part_step + attn_part_row(g, bh, row, token, hq);
        if (half == 0) *(attn_f32x2 *)(g.part_ml + at * 2) = attn_f32x2{m, l};
        if (l != 0.0f)  // (true of NaN) nothing seen: nothing is read there
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    attn_store4<PT_FLOAT32>(g.part_o + at * g.size, d * 32 + 8 * e + 4 * half, g.size, o[d][4 * e],
                                            o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]);
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const long long to = b * g.o_bs + token * g.o_ts + hq * g.o_hs;
#pragma unroll
    for (int d = 0; d < ND; d++) {
        attn_store_block<DT>((typename AttnT<DT>::S *)g.out + to, d * 32, g.size, half, [&](int r) { return o[d][r] * inv; });
        if constexpr (DT != PT_FLOAT32) {
            if (g.rest)
                attn_store_block<DT>((typename AttnT<DT>::S *)g.rest + to, d * 32, g.size, half,
                                     [&](int r) { return attn_rest<DT>(o[d][r] * inv); });
        }
    }
    if (g.lse && half == 0)
        g.lse[(g.q_starts ? 0 : (long long)b * g.heads * g.nq) + (long long)hq * g.stat_rows + (g.q_starts ? token : qi)] =
            l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
}

// ------------------------------------------------------------- forward
// Rows of a key head are its queries times its `group` query heads, row r =
// query r / group, head r % group, so that the heads that share keys share
// the staged tiles, and a single token's heads fill a block together.
//
// Four waves of 32 rows each read every staged tile of keys and values.  The
// scores of tile t + 1 are computed beside the exponentials of tile t, and
// the maximum of those scores beside the product of tile t with its values,
// so that the matrix and the vector pipe of a SIMD run together also inside
// one wave: one tile takes 1024 cycles of MFMA and about as many of vector
// instructions (half of them exponentials, at a quarter of the rate).  Issue
// of both pipes and the clock under this load bound it (MFMA busy 50 %; taking
// any one part away saves 4 to 17 %): six causal prompts of 1 to 4096 tokens,
// 16 heads of 128 in bfloat16, 140 to 149 us on different cards, 910 to 975
// TFLOP/s.
template <int DT, int DP> struct AttnFwdShape {
    static constexpr int ES = AttnT<DT>::ES;
    static constexpr int BN = ES == 4 || DP == 256 ? 32 : 64;
    static constexpr int WGS = 4 * attn_tile_bytes(BN, DP, ES) <= 65536 && DP <= 128 ? 2 : 1;
    static_assert(4 * attn_tile_bytes(BN, DP, ES) <= 131072, "two buffers of keys and values");
};

template <int DT, int DP, bool VEC>
__global__ __launch_bounds__(256, (AttnFwdShape<DT, DP>::WGS)) void k_attention(AttnArgs g)
{
    using T = AttnT<DT>;
    using S = typename T::S;
    constexpr int BN = AttnFwdShape<DT, DP>::BN, NKB = BN / 32, BM = 128;
    constexpr int KS = DP * T::ES / 32, ND = DP / 32;
    __shared__ __attribute__((aligned(1024))) S k0[BN * DP], v0[BN * DP], k1[BN * DP], v1[BN * DP];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int split = blockIdx.y;
    int tile, bh;
    if (!attn_place(g, false, tile, bh)) return;  // whole workgroup
    const int b = bh / g.kv_heads, hk = bh % g.kv_heads;
    const AttnSeq sq = attn_seq(g.q_starts, g.q_lengths, g.q_rows, g.nq, b);
    const AttnSeq sk = attn_seq(g.k_starts, g.k_lengths, g.k_rows, g.nk, b);
    const int rows = sq.n * g.group, row0 = tile * BM;
    if (row0 >= rows) return;  // whole workgroup
    const int row = row0 + wave * 32 + (lane & 31), qi = row / g.group, hq = hk * g.group + row % g.group;
    const bool live = row < rows;

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
    auto load_k = [&](int t, S *to) { kl.load(ks, g.size, t * BN, to, wave, lane); };
    auto load_v = [&](int t, S *to) { vl.load(vs, g.size, t * BN, to, wave, lane); };
    if (t0 < t1) load_k(t0, k0);

    typename T::Frag q[KS];
    attn_row<DT, DP, VEC>(q, (const S *)g.q + b * g.q_bs + (sq.row + qi) * g.q_ts + hq * g.q_hs, live, g.size, half);
    float m = -INFINITY, l = 0.0f;
    floatx16 o[ND], sa[NKB], sb[NKB];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] = 0.0f;
    AttnLane<DT, DP> at;
    at.init(lane);

    auto scores = [&](const S *kt, floatx16 (&s)[NKB]) {
#pragma unroll
        for (int kb = 0; kb < NKB; kb++) s[kb] = attn_rows<DT, DP>(kt, kb * 32, q, at);
    };
    auto mask = [&](int t, floatx16 (&s)[NKB]) {
        if ((t + 1) * BN <= lim_first) return;  // uniform: every row sees every key
        const int key0 = t * BN + 4 * half;
#pragma unroll
        for (int kb = 0; kb < NKB; kb++)
#pragma unroll
            for (int r = 0; r < 16; r++) s[kb][r] = key0 + kb * 32 + 8 * (r / 4) + r % 4 < lim ? s[kb][r] : -INFINITY;
    };
    auto maximum = [&](const floatx16 (&s)[NKB]) {
        float top = s[0][0];
#pragma unroll
        for (int kb = 0; kb < NKB; kb++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[kb][r]);
        return fmaxf(top, attn_other(top, lane)) * g.scale_log2;
    };
    // The reference m of the exponentials follows the maximum only when it is
    // passed by more than 8 (a factor of 256): sums and products are fp32 and
    // a probability keeps its relative precision whatever its size, so most
    // tiles need no rescaling of the sums.
    bool far = false;
    auto follow = [&](float top) {
        if (__all(!(top > m + 8.0f))) return;
        const float to = fmaxf(m, top), a = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
        far = far || __any(attn_far(to));
        m = to;
        l *= a;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[d][e] *= a;
    };
    // one exponential of the tile, register e
    auto exponential = [&](floatx16 (&s)[NKB], int e, float ref) {
        float x = __builtin_amdgcn_exp2f(fmaf(s[e / 16][e % 16], g.scale_log2, -ref));
        asm volatile("" : "+v"(x));  // here, beside the products, and not where it is used
        s[e / 16][e % 16] = x;
        l += x;
    };
    constexpr int NU = NKB * KS, NP = attn_col_units<DT, DP>(), AHEAD = 2;
    // tile t, whose scores are `now`: the next tile's keys lie in kn, those
    // after them go to kf, this tile's values lie in vt, the next go to vn
    auto step = [&](int t, floatx16 (&now)[NKB], floatx16 (&next)[NKB], const S *kn, S *kf, const S *vt, S *vn, auto MORE) {
        constexpr bool more = decltype(MORE)::value;  // there is a next tile
        attn_landed();
        at.fresh();
        if constexpr (more) {
            if (t + 2 < t1) load_k(t + 2, kf);
            load_v(t + 1, vn);
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        // the next scores, beside the first block's exponentials
        if constexpr (more) {
            typename T::Frag f[AHEAD + 1];
#pragma unroll
            for (int u = 0; u < AHEAD; u++) f[u] = attn_row_frag<DT, DP>(kn, u / KS * 32, u % KS, at);
#pragma unroll
            for (int kb = 0; kb < NKB; kb++)
#pragma unroll
                for (int e = 0; e < 16; e++) next[kb][e] = 0.0f;
            static_for<0, NU>([&](auto U) {
                constexpr int u = decltype(U)::value, w = u + AHEAD;
                if constexpr (w < NU) f[w % (AHEAD + 1)] = attn_row_frag<DT, DP>(kn, w / KS * 32, w % KS, at);
                attn_mfma<DT>(next[u / KS], f[u % (AHEAD + 1)], q[u % KS]);
                static_for<u * 16 / NU, (u + 1) * 16 / NU>([&](auto E) { exponential(now, decltype(E)::value, ref); });
                __builtin_amdgcn_sched_barrier(0);
            });
        } else {
            static_for<0, 16>([&](auto E) { exponential(now, decltype(E)::value, ref); });
        }
        if constexpr (more) mask(t + 1, next);
        // the product with the values, beside the second block's
        // exponentials and, last, the next scores' maximum
        float top = -INFINITY;
        static_for<0, NKB>([&](auto KB) {
            constexpr int kb = decltype(KB)::value;
            AttnColFrag<DT> f[AHEAD + 1], right;
#pragma unroll
            for (int u = 0; u < AHEAD; u++) f[u] = attn_col_frag<DT, DP>(vt, kb * 32, u, at);
            static_for<0, NP>([&](auto U) {
                constexpr int u = decltype(U)::value, w = u + AHEAD;
                if constexpr (w < NP) f[w % (AHEAD + 1)] = attn_col_frag<DT, DP>(vt, kb * 32, w, at);
                if constexpr (u % ND == 0) right = attn_col_right<DT, DP>(now[kb], u);
                attn_col_mfma<DT, DP>(o, u, f[u % (AHEAD + 1)], right);
                if constexpr (kb + 1 < NKB) {
                    static_for<u * 16 / NP, (u + 1) * 16 / NP>([&](auto E) { exponential(now, 16 + decltype(E)::value, ref); });
                } else if constexpr (more) {
                    static_for<u * NKB * 16 / NP, (u + 1) * NKB * 16 / NP>([&](auto E) {
                        constexpr int e = decltype(E)::value;
                        top = fmaxf(top, next[e / 16][e % 16]);
                    });
                    asm volatile("" : "+v"(top));
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        });
        if constexpr (more) follow(fmaxf(top, attn_other(top, lane)) * g.scale_log2);
    };
    if (t0 < t1) {
        attn_landed();
        if (t0 + 1 < t1) load_k(t0 + 1, k1);
        load_v(t0, v0);
        scores(k0, sa);
        mask(t0, sa);
        follow(maximum(sa));
    }
    int t = t0;
    for (; t + 2 < t1; t += 2) {
        step(t, sa, sb, k1, k0, v0, v1, std::true_type{});
        step(t + 1, sb, sa, k0, k1, v1, v0, std::true_type{});
    }
    if (t + 1 < t1) {
        step(t, sa, sb, k1, k0, v0, v1, std::true_type{});
        step(t + 1, sb, sa, k0, k1, v1, v0, std::false_type{});
    } else if (t < t1) {
        step(t, sa, sb, k1, k0, v0, v1, std::false_type{});
    }
    if (__builtin_expect(attn_any_wave<4>(far, lane, wave), 0)) {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[d][e] = 0.0f;
        for (t = t0; t < t1; t++) {
            __syncthreads();
            load_k(t, k0);
            load_v(t, v0);
            attn_landed();
#pragma unroll 1
            for (int kb = 0; kb < NKB; kb++) {
                at.fresh();
                floatx16 s = attn_rows<DT, DP>(k0, kb * 32, q, at);
#pragma unroll
                for (int r = 0; r < 16; r++) s[r] = t * BN + kb * 32 + 4 * half + 8 * (r / 4) + r % 4 < lim ? s[r] : -INFINITY;
                attn_far_block<DT, DP>(s, m, l, o, g.scale_log2, v0, kb * 32, at, lane);
            }
        }
        attn_far_part<ND>(m, l, o, g.scale_log2, g.splits > 1);
    }
    l += attn_other(l, lane);
    // the row's numbers once more, so that no register holds them in the loops
    int at_row = row0 + wave * 32 + (lane & 31);
    asm volatile("" : "+v"(at_row));
    const int token = at_row / g.group;
    attn_result<DT, ND>(g, m, l, o, at_row < rows, b, bh, at_row, sq.row + token, token, hk * g.group + at_row % g.group, split, half);
}

// 32 rows or fewer, rows of whole 16-byte packs: single tokens over a cache,
// bound by reading keys and values.  Each wave walks key blocks of 32 of its
// own, every NW-th of the range, through a block of LDS of its own: no
// barrier, and the waves drift apart, so that loads are on their way at all
// times.  The next block's loads go to registers while this one is computed.
// 32 caches of 977 to 8076 tokens, 8 key heads of 128 in bfloat16, 594 MB:
// 107 to 112 us (5.3 to 5.5 TB/s) and 5.4 us for the join of the ranges.
template <int DT, int DP> struct AttnTokenShape {
    static constexpr int TILE = attn_tile_bytes(32, DP, AttnT<DT>::ES);
    static constexpr int NW = TILE <= 8192 ? 4 : TILE <= 16384 ? 2 : 1;
    static constexpr int WGS = TILE <= 8192 ? 2 : 1;  // waves per SIMD that the registers are kept for
};

template <int DT, int DP>
__global__ __launch_bounds__((64 * AttnTokenShape<DT, DP>::NW), (AttnTokenShape<DT, DP>::WGS))
void k_attention_token(AttnArgs g)
{
    using T = AttnT<DT>;
    using S = typename T::S;
    constexpr int NW = AttnTokenShape<DT, DP>::NW, TE = 32 * DP;
    constexpr int KS = DP * T::ES / 32, ND = DP / 32, NI = TE * T::ES / 1024;
    __shared__ __attribute__((aligned(1024))) S kt[NW * TE], vt[NW * TE];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int split = blockIdx.y;
    const int bh = (int)blockIdx.x, b = bh / g.kv_heads, hk = bh % g.kv_heads;
    const AttnSeq sq = attn_seq(g.q_starts, g.q_lengths, g.q_rows, g.nq, b);
    const AttnSeq sk = attn_seq(g.k_starts, g.k_lengths, g.k_rows, g.nk, b);
    const int rows = sq.n * g.group, row = lane & 31;
    if (!rows) return;  // whole workgroup
    const int qi = row / g.group, hq = hk * g.group + row % g.group;
    const bool live = row < rows;

    const AttnSrc ks = {(const char *)((const S *)g.k + b * g.k_bs + sk.row * g.k_ts + hk * g.k_hs), g.k_ts * T::ES, sk.n};
    const AttnSrc vs = {(const char *)((const S *)g.v + b * g.v_bs + sk.row * g.v_ts + hk * g.v_hs), g.v_ts * T::ES, sk.n};
    AttnStage<DT, DP, 32, 1, true> kl, vl;
    kl.init(ks, g.size, 0, lane);
    vl.init(vs, g.size, 0, lane);
    const int shift = sk.n - sq.n + 1, last = g.causal ? min(sk.n, (rows - 1) / g.group + shift) : sk.n;
    const int lim = g.causal ? min(sk.n, qi + shift) : sk.n, lim_first = g.causal ? min(sk.n, shift) : sk.n;
    // this range's blocks, every NW-th of them for this wave
    const int blocks = max(0, (last + 31) / 32), per = (((sk.n + 31) / 32 + g.splits - 1) / g.splits + NW - 1) / NW * NW;
    const int t1 = min(blocks, per * (split + 1)), t0 = per * split + wave;

    S *const kw = kt + wave * TE, *const vw = vt + wave * TE;
    floatx4 kr[NI], vr[NI];
    if (t0 < t1) {
        kl.fetch(ks, g.size, t0 * 32, kr);
        vl.fetch(vs, g.size, t0 * 32, vr);
    }
    typename T::Frag q[KS];
    attn_row<DT, DP, true>(q, (const S *)g.q + b * g.q_bs + (sq.row + qi) * g.q_ts + hq * g.q_hs, live, g.size, half);
    float m = -INFINITY, l = 0.0f;
    floatx16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] = 0.0f;
    AttnLane<DT, DP> at;
    at.init(lane);
    bool far = false;
    for (int t = t0; t < t1; t += NW) {
        at.fresh();
#pragma unroll
        for (int i = 0; i < NI; i++) *(floatx4 *)(kw + (i * 64 + lane) * T::PK) = kr[i];
#pragma unroll
        for (int i = 0; i < NI; i++) *(floatx4 *)(vw + (i * 64 + lane) * T::PK) = vr[i];
        if (t + NW < t1) {
            kl.fetch(ks, g.size, (t + NW) * 32, kr);
            vl.fetch(vs, g.size, (t + NW) * 32, vr);
        }
        floatx16 s = attn_rows<DT, DP>(kw, 0, q, at);
        const int key0 = t * 32 + 4 * half;
        if ((t + 1) * 32 > lim_first) {
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = key0 + 8 * (r / 4) + r % 4 < lim ? s[r] : -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int r = 1; r < 16; r++) top = fmaxf(top, s[r]);
        top = fmaxf(top, attn_other(top, lane)) * g.scale_log2;
        if (!__all(!(top > m + 8.0f))) {  // as in k_attention
            const float to = fmaxf(m, top), a = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
            far = far || __any(attn_far(to));
            m = to;
            l *= a;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[d][e] *= a;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], g.scale_log2, -ref));
            l += s[r];
        }
        attn_cols<DT, DP>(o, vw, 0, s, at);
    }
    const bool again = NW > 1 ? attn_any_wave<NW>(far, lane, wave) : far;
    if (__builtin_expect(again, 0)) {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[d][e] = 0.0f;
        for (int t = t0; t < t1; t += NW) {
            kl.fetch(ks, g.size, t * 32, kr);
            vl.fetch(vs, g.size, t * 32, vr);
#pragma unroll
            for (int i = 0; i < NI; i++) *(floatx4 *)(kw + (i * 64 + lane) * T::PK) = kr[i];
#pragma unroll
            for (int i = 0; i < NI; i++) *(floatx4 *)(vw + (i * 64 + lane) * T::PK) = vr[i];
            at.fresh();
            floatx16 s = attn_rows<DT, DP>(kw, 0, q, at);
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = t * 32 + 4 * half + 8 * (r / 4) + r % 4 < lim ? s[r] : -INFINITY;
            attn_far_block<DT, DP>(s, m, l, o, g.scale_log2, vw, 0, at, lane);
        }
        if (NW > 1) __syncthreads();
    }

    l += attn_other(l, lane);
    if constexpr (NW > 1) {
        attn_join_waves<NW, ND>(m, l, o, again ? g.scale_log2 : 1.0f, (float *)kt, lane, wave);
        static_assert(NW * 1024 * 4 <= NW * TE * T::ES, "the joined block fits a tile");
        if (wave) return;
    }
    if (again) attn_far_part<ND>(m, l, o, g.scale_log2, g.splits > 1);
    // the row's numbers once more, as in k_attention
    int at_row = lane & 31;
    asm volatile("" : "+v"(at_row));
    const int token = at_row / g.group;
    attn_result<DT, ND>(g, m, l, o, at_row < rows, b, bh, at_row, sq.row + token, token, hk * g.group + at_row % g.group, split, half);
}

// ------------------------------------------- gradient of keys and values
// A wave keeps 32 keys and their values and streams the queries that see
// them, head by head of the group, so the sum over heads that share a key
// stays in its registers and no order of additions can change.
//
// Blocks of 32 queries go through a pipeline of two: the scores and the
// products with the values of block i + 1 run on the matrix pipe beside the
// exponentials and differences of block i, then come block i's two products
// into the sums.  The tiles lie in three buffers, since block i + 1 may be
// the next tile's: one barrier a tile, and a tile has the time of a whole one
// to arrive.  4 x 2048 causal tokens, 16 heads of 128 over 8 key heads in
// bfloat16: 180 us at the highest clock, where it took 232 without the
// pipeline (MFMA busy 40 %, 760 TFLOP/s of the four products; up to 199 on
// cards that clock lower under it); one wave a SIMD, since the two sums and
// the two rows take 320 registers.
//
// PASS 0 computes both gradients.  Heads past 128 elements, whose rows and
// sums together would pass the register file, take PASS 1 (values) and PASS 2
// (keys).
template <int DT, int DP> struct AttnBwdShape {
    static constexpr int ES = AttnT<DT>::ES;
    static constexpr int BQ = ES == 4 || DP == 256 ? 32 : 64;  // queries of a tile, keys' gradient
    static constexpr int BN = BQ;                              // keys of a tile, queries' gradient
    static constexpr int NBUF = 6 * attn_tile_bytes(BQ, DP, ES) <= 131072 ? 3 : 2;
    static constexpr int KWGS = DP <= 64 ? 2 : 1;              // workgroups a CU
    static constexpr int QWGS = DP * ES <= 256 ? 2 : 1;
    static constexpr bool kSplitPasses = DP == 256;
};

// Four bytes a lane into LDS, zeros past `range`.
__device__ __forceinline__ void attn_load_lds4(const void *base, uint32_t off, float *lds, uint32_t range)
{
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)range, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (PT_LDS_AS void *)lds, 4, off, 0, 0, 0);
}

template <int DT, int DP, int PASS, bool VEC>
__global__ __launch_bounds__(256, (AttnBwdShape<DT, DP>::KWGS)) void k_attention_dkv(AttnArgs g)
{
    using T = AttnT<DT>;
    using S = typename T::S;
    constexpr int BQ = AttnBwdShape<DT, DP>::BQ, NQB = BQ / 32, KS = DP * T::ES / 32, ND = DP / 32, TE = BQ * DP;
    constexpr int NBUF = AttnBwdShape<DT, DP>::NBUF;
    constexpr int AHEAD = AttnBwdShape<DT, DP>::KWGS == 1 ? 6 : 3, NCOL = attn_col_units<DT, DP>();
    constexpr bool kV = PASS != 2, kK = PASS != 1;
    // queries, then upstream gradients; lse, the rows' sums, what their scores lose
    __shared__ __attribute__((aligned(1024))) S b0[2 * TE], b1[2 * TE], b2[NBUF == 3 ? 2 * TE : 8];
    __shared__ __attribute__((aligned(256))) float s0[192], s1[192], s2[192];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    int tile, bh;
    if (!attn_place(g, true, tile, bh)) return;  // whole workgroup
    const int b = bh / g.kv_heads, hk = bh % g.kv_heads;
    const AttnSeq sq = attn_seq(g.q_starts, g.q_lengths, g.q_rows, g.nq, b);
    const AttnSeq sk = attn_seq(g.k_starts, g.k_lengths, g.k_rows, g.nk, b);
    const int first = tile * 128;
    if (first >= sk.n) return;  // whole workgroup
    const int key = first + wave * 32 + (lane & 31);
    const bool live = key < sk.n;

    // query i sees key j where i >= j - shift
    const int shift = sk.n - sq.n;
    const int from = g.causal ? key - shift : INT_MIN;
    const int t0 = g.causal ? max(0, first - shift) / BQ : 0, per = max(0, (sq.n + BQ - 1) / BQ - t0);
    // this workgroup's share of the tiles of all heads
    const int share = (per * g.group + g.splits - 1) / g.splits;
    const int step0 = share * (int)blockIdx.y, steps = min(per * g.group, step0 + share);

    const S *qb = (const S *)g.q + b * g.q_bs + sq.row * g.q_ts, *wb = (const S *)g.w + b * g.o_bs + sq.row * g.o_ts;
    const long long stat = g.q_starts ? sq.row : (long long)b * g.heads * g.nq;
    AttnStage<DT, DP, BQ, 4, VEC> ql, wl;
    ql.init({nullptr, g.q_ts * T::ES, 0}, g.size, wave, lane);
    wl.init({nullptr, g.o_ts * T::ES, 0}, g.size, wave, lane);
    auto load = [&](int it, S *to, float *st) __attribute__((always_inline)) {
        const int hq = hk * g.group + it / per, r0 = (t0 + it % per) * BQ;
        ql.load({(const char *)(qb + hq * g.q_hs), g.q_ts * T::ES, sq.n}, g.size, r0, to, wave, lane);
        wl.load({(const char *)(wb + hq * g.o_hs), g.o_ts * T::ES, sq.n}, g.size, r0, to + TE, wave, lane);
        const long long at = stat + (long long)hq * g.stat_rows + r0;
        const uint32_t range = (uint32_t)min(sq.n - r0, BQ) * 4u;
        // rows past the last have zero products; a zero lse keeps their exponentials finite
        if (wave == 0) attn_load_lds4(g.lse2 + at, lane * 4u, st, range);
        if (wave == 1) attn_load_lds4(g.delta + at, lane * 4u, st + 64, range);
        if (wave == 2) attn_load_lds4(g.tops + at, lane * 4u, st + 128, range);
    };
    if (step0 < steps) {
        load(step0, b0, s0);
        if (step0 + 1 < steps) load(step0 + 1, b1, s1);
    }
    typename T::Frag k[KS], v[kK ? KS : 1];
    attn_row<DT, DP, VEC>(k, (const S *)g.k + b * g.k_bs + (sk.row + key) * g.k_ts + hk * g.k_hs, live, g.size, half);
    if constexpr (kK)
        attn_row<DT, DP, VEC>(v, (const S *)g.v + b * g.v_bs + (sk.row + key) * g.v_ts + hk * g.v_hs, live, g.size, half);
    floatx16 dk[ND], dv[ND], pa, pb, ta, tb;
#pragma unroll
    for (int e = 0; e < 16; e++) {
#pragma unroll
        for (int d = 0; d < ND; d++) dk[d][e] = dv[d][e] = 0.0f;
    }
    AttnLane<DT, DP> at;
    at.init(lane);
    auto of_key = [&](int f) { return k[f]; };
    auto of_value = [&](int f) { return v[kK ? f : 0]; };
    auto nothing = [](auto, auto) {};
    // block qi of the tile in `now`, step `it`; the next block lies in `next` from row `row`
    auto block = [&](int it, int qi, floatx16 &p, floatx16 &t, floatx16 &pn, floatx16 &tn, const S *now, const float *st,
                     const S *next, int row) __attribute__((always_inline)) {
        at.fresh();
        floatx4 ls[4], es[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            ls[r] = *(const floatx4 *)(st + qi * 32 + 8 * r + 4 * half);
            if constexpr (kK) es[r] = *(const floatx4 *)(st + 64 + qi * 32 + 8 * r + 4 * half);
        }
        // (looked at here and not once for all queries: 2 us of 180 instead of 6; these scores' product ended a block
        // ago, so nothing has to wait for it behind the branch)
        if (__builtin_expect(__any(st[128 + qi * 32 + (lane & 31)] != 0.0f), 0)) {
#pragma unroll
            for (int r = 0; r < 16; r++) p[r] -= st[128 + qi * 32 + 8 * (r / 4) + 4 * half + r % 4];
        }
        // the next block's scores beside this one's exponentials, its products
        // with the values beside the differences, then this block's sums
        constexpr int NA = KS, NB = NA + (kK ? KS : 0), NC = NB + (kV ? NCOL : 0), N = NC + (kK ? NCOL : 0);
        AttnColFrag<DT> right[NCOL / ND];
#pragma unroll
        for (int e = 0; e < 16; e++) pn[e] = tn[e] = 0.0f;
        attn_queue<DT, N, AHEAD>(
            [&](auto I) __attribute__((always_inline)) {
                constexpr int u = decltype(I)::value;
                if constexpr (u < NA) return attn_row_frag<DT, DP>(next, row, u, at);
                else if constexpr (u < NB) return attn_row_frag<DT, DP>(next + TE, row, u - NA, at);
                else if constexpr (u < NC) return attn_any<DT>(attn_col_frag<DT, DP>(now + TE, qi * 32, u - NB, at));
                else return attn_any<DT>(attn_col_frag<DT, DP>(now, qi * 32, u - NC, at));
            },
            [&](auto I, const typename T::Frag &f) __attribute__((always_inline)) {
                constexpr int u = decltype(I)::value;
                // (asm: here, beside the products, and not where they are used)
                if constexpr (u < NA) {
                    attn_mfma<DT>(pn, f, k[u]);
                    attn_share(IC<u>{}, IC<NA>{}, [&](int r) {
                        float x = __builtin_amdgcn_exp2f(fmaf(p[r], g.scale_log2, -ls[r / 4][r % 4]));
                        asm volatile("" : "+v"(x));
                        p[r] = x;
                    });
                    if constexpr (u + 1 == NA) {
                        const int r0 = (t0 + it % per) * BQ;
                        if (g.causal && r0 < first + 127 - shift) {
                            const int i0 = r0 + qi * 32 + 4 * half;
#pragma unroll
                            for (int r = 0; r < 16; r++) p[r] = i0 + 8 * (r / 4) + r % 4 >= from ? p[r] : 0.0f;
                        }
                    }
                } else if constexpr (u < NB) {
                    attn_mfma<DT>(tn, f, v[kK ? u - NA : 0]);
                    attn_share(IC<u - NA>{}, IC<KS>{}, [&](int r) {
                        float x = p[r] * (t[r] - es[r / 4][r % 4]);
                        asm volatile("" : "+v"(x));
                        t[r] = x;
                    });
                } else if constexpr (u < NC) {
                    if constexpr ((u - NB) % ND == 0) right[(u - NB) / ND] = attn_col_right<DT, DP>(p, u - NB);
                    attn_col_mfma<DT, DP>(dv, u - NB, attn_of_any<DT>(f), right[(u - NB) / ND]);
                } else {
                    if constexpr ((u - NC) % ND == 0) right[(u - NC) / ND] = attn_col_right<DT, DP>(t, u - NC);
                    attn_col_mfma<DT, DP>(dk, u - NC, attn_of_any<DT>(f), right[(u - NC) / ND]);
                }
            });
    };
    // a step: its tile lies in `now`, the next in `next`, the one after goes to `later`
    auto step = [&](int it, floatx16 &p, floatx16 &t, floatx16 &pn, floatx16 &tn, S *now, float *st, S *next, S *later, float *sl) __attribute__((always_inline)) {
        if constexpr (NQB == 2) block(it, 0, p, t, pn, tn, now, st, now, 32);
        attn_landed();  // the next tile is there, and every wave is done with the one before this
        if (NBUF == 3 && it + 2 < steps) load(it + 2, later, sl);
        // (after the last tile the next block is computed from what lies there, and used by nobody)
        if constexpr (NQB == 2) block(it, 1, pn, tn, p, t, now, st, next, 0);
        else block(it, 0, p, t, pn, tn, now, st, next, 0);
        if constexpr (NBUF == 2) {
            attn_landed();
            if (it + 2 < steps) load(it + 2, now, st);
        }
    };
    if (step0 < steps) {
        attn_landed();
        at.fresh();
        attn_rows_beside<DT, DP, AHEAD>(pa, b0, 0, of_key, at, nothing);
        if constexpr (kK) attn_rows_beside<DT, DP, AHEAD>(ta, b0 + TE, 0, of_value, at, nothing);
    }
    // with one block a tile the two score registers change places from step to step
    auto steps_of = [&](int it, floatx16 &p, floatx16 &t, floatx16 &pn, floatx16 &tn, auto TURN) __attribute__((always_inline)) {
        constexpr int n = decltype(TURN)::value % NBUF;
        if constexpr (NBUF == 2) {
            if constexpr (n == 0) step(it, p, t, pn, tn, b0, s0, b1, b0, s0);
            else step(it, p, t, pn, tn, b1, s1, b0, b1, s1);
        } else if constexpr (n == 0) {
            step(it, p, t, pn, tn, b0, s0, b1, b2, s2);
        } else if constexpr (n == 1) {
            step(it, p, t, pn, tn, b1, s1, b2, b0, s0);
        } else {
            step(it, p, t, pn, tn, b2, s2, b0, b1, s1);
        }
    };
    constexpr int TURNS = NQB == 2 ? NBUF : NBUF == 3 ? 6 : 2;
    for (int it = step0; it < steps; it += TURNS)
        static_for<0, TURNS>([&](auto TURN) __attribute__((always_inline)) {
            constexpr int n = decltype(TURN)::value;
            if (it + n < steps) {
                if constexpr (NQB == 2 || n % 2 == 0) steps_of(it + n, pa, ta, pb, tb, TURN);
                else steps_of(it + n, pb, tb, pa, ta, TURN);
            }
        });
    if (!live) return;
    // gradients are contiguous, and so is each share's part of them
    const long long to = ((g.k_starts ? sk.row + key : (long long)b * g.nk + key) * g.kv_heads + hk) * g.size;
#pragma unroll
    for (int d = 0; d < ND; d++) {
        auto put = [&](void *whole, float *part, const floatx16 &x, float c) {
            auto value = [&](int r) { return x[r] * c; };
            if (g.splits > 1) attn_store_block<PT_FLOAT32>(part + blockIdx.y * g.part_step + to, d * 32, g.size, half, value);
            else attn_store_block<DT>((S *)whole + to, d * 32, g.size, half, value);
        };
        if constexpr (kV) put(g.dv, g.part_ml, dv[d], 1.0f);
        if constexpr (kK) put(g.dk, g.part_o, dk[d], g.scale);
    }
}

// Rows whose lse is farther from 0 than this have it computed anew by the
// queries' gradient, as the largest score and the sum of exponentials beside
// it: p = 2^(c s - lse2) is off by the rounding of lse, 2^-24 of it, in every
// element of the row (6e-5 at 512, everything at 1e9).
constexpr float kExactLse = 512.0f;

// ------------------------------------------------- gradient of the queries
// Rows as in the forward pass; the keys and values stream past them.  This
// pass runs first and leaves lse2 and d for the other: it holds w anyway.  Two
// workgroups a CU run beside each other's waits where the registers allow it:
// 134 us for the tokens above at the highest clock, 147 in the middle, against
// 160 with one; reading further ahead spilled (158 and 173 us).
template <int DT, int DP, bool VEC>
__global__ __launch_bounds__(256, (AttnBwdShape<DT, DP>::QWGS)) void k_attention_dq(AttnArgs g)
{
    using T = AttnT<DT>;
    using S = typename T::S;
    constexpr int BN = AttnBwdShape<DT, DP>::BN, NKB = BN / 32, KS = DP * T::ES / 32, ND = DP / 32, BM = 128;
    __shared__ __attribute__((aligned(1024))) S k0[BN * DP], v0[BN * DP], k1[BN * DP], v1[BN * DP];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    int tile, bh;
    if (!attn_place(g, false, tile, bh)) return;  // whole workgroup
    const int b = bh / g.kv_heads, hk = bh % g.kv_heads;
    const AttnSeq sq = attn_seq(g.q_starts, g.q_lengths, g.q_rows, g.nq, b);
    const AttnSeq sk = attn_seq(g.k_starts, g.k_lengths, g.k_rows, g.nk, b);
    const int rows = sq.n * g.group, row0 = tile * BM;
    if (row0 >= rows) return;  // whole workgroup
    const int row = row0 + wave * 32 + (lane & 31), qi = row / g.group, hq = hk * g.group + row % g.group;
    const bool live = row < rows;

    typename T::Frag q[KS], w[KS];
    attn_row<DT, DP, VEC>(q, (const S *)g.q + b * g.q_bs + (sq.row + qi) * g.q_ts + hq * g.q_hs, live, g.size, half);
    attn_row<DT, DP, VEC>(w, (const S *)g.w + b * g.o_bs + (sq.row + qi) * g.o_ts + hq * g.o_hs, live, g.size, half);
    const long long stat0 = g.q_starts ? sq.row : (long long)b * g.heads * g.nq, stat = stat0 + (long long)hq * g.stat_rows + qi;
    // d in fp32, of the output as it was before its rounding where that is
    // known; a row that sees no key gets lse +inf, so its exponentials are 0
    float es = 0.0f, ls = INFINITY, lost = 0.0f;
    bool far = false;
    {
        typename T::Frag o[KS];
        const long long from = b * g.o_bs + (sq.row + qi) * g.o_ts + hq * g.o_hs;
        attn_row<DT, DP, VEC>(o, (const S *)g.out + from, live, g.size, half);
#pragma unroll
        for (int f = 0; f < KS; f++) es = attn_dot<DT>(w[f], o[f], es);
        if (DT != PT_FLOAT32 && g.rest) {
            attn_row<DT, DP, VEC>(o, (const S *)g.rest + from, live, g.size, half);
#pragma unroll
            for (int f = 0; f < KS; f++) es = attn_dot<DT>(w[f], o[f], es);
        }
        es += attn_other(es, lane);
        if (live) {
            const float l = g.lse[stat];
            if (l != -INFINITY) ls = l * 1.4426950408889634f;
            far = l != -INFINITY && fabsf(l) > kExactLse;
        }
    }

    const AttnSrc ks = {(const char *)((const S *)g.k + b * g.k_bs + sk.row * g.k_ts + hk * g.k_hs), g.k_ts * T::ES, sk.n};
    const AttnSrc vs = {(const char *)((const S *)g.v + b * g.v_bs + sk.row * g.v_ts + hk * g.v_hs), g.v_ts * T::ES, sk.n};
    AttnStage<DT, DP, BN, 4, VEC> kl, vl;
    kl.init(ks, g.size, wave, lane);
    vl.init(vs, g.size, wave, lane);
    const int shift = sk.n - sq.n + 1;
    const int lim = g.causal ? min(sk.n, qi + shift) : sk.n;
    const int lim_first = g.causal ? min(sk.n, row0 / g.group + shift) : sk.n;
    const int lim_last = g.causal ? min(sk.n, (min(row0 + BM, rows) - 1) / g.group + shift) : sk.n;
    // this workgroup's share of the sequence's key tiles
    const int share = ((sk.n + BN - 1) / BN + g.splits - 1) / g.splits, t0 = share * (int)blockIdx.y;
    const int tiles = max(0, (lim_last + BN - 1) / BN);
    int t1 = min(tiles, t0 + share);
    AttnLane<DT, DP> at;
    at.init(lane);

    // every wave looks at the rows of all four, for the barriers
    bool some = false;
    for (int r = row0 + lane; r < min(row0 + BM, rows); r += 64) {
        const float l = g.lse[stat0 + (long long)(hk * g.group + r % g.group) * g.stat_rows + r / g.group];
        some = some || (l != -INFINITY && fabsf(l) > kExactLse);
    }
    const bool exact = __any(some);
    if (__builtin_expect(exact, 0)) {
        float m = -INFINITY, l = 0.0f;
        for (int t = 0; t < tiles; t++) {
            __syncthreads();
            kl.load(ks, g.size, t * BN, k0, wave, lane);
            attn_landed();
            at.fresh();
#pragma unroll 1
            for (int kb = 0; kb < NKB; kb++) {
                floatx16 s = attn_rows<DT, DP>(k0, kb * 32, q, at);
                float top = m;
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    s[r] = t * BN + kb * 32 + 4 * half + 8 * (r / 4) + r % 4 < lim ? s[r] : -INFINITY;
                    top = fmaxf(top, s[r]);
                }
                const float from = top == -INFINITY ? 0.0f : top;
                l *= __builtin_amdgcn_exp2f((m - from) * g.scale_log2);
                m = top;
#pragma unroll
                for (int r = 0; r < 16; r++) l += __builtin_amdgcn_exp2f((s[r] - from) * g.scale_log2);
            }
        }
        // the two lanes of a row
        const float m2 = attn_other(m, lane), l2 = attn_other(l, lane), top = fmaxf(m, m2);
        l = l * __builtin_amdgcn_exp2f((m - top) * g.scale_log2) + l2 * __builtin_amdgcn_exp2f((m2 - top) * g.scale_log2);
        if (far) {
            lost = top;
            ls = __builtin_amdgcn_logf(l);
        }
    }
    if (live && blockIdx.y == 0 && half == 0) {
        g.lse2[stat] = ls;
        g.delta[stat] = es;
        g.tops[stat] = lost;
    }

    floatx16 dq[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) dq[d][e] = 0.0f;
    // These workgroups go through their tiles here, without the loop below.  (In that loop the difference would be a
    // branch behind the scores' product, and for such a branch the compiler left out the waits for the product.)
    if (__builtin_expect(exact, 0)) {
        for (int t = t0; t < t1; t++) {
            __syncthreads();
            kl.load(ks, g.size, t * BN, k0, wave, lane);
            vl.load(vs, g.size, t * BN, v0, wave, lane);
            attn_landed();
#pragma unroll 1
            for (int kb = 0; kb < NKB; kb++) {
                at.fresh();
                floatx16 p = attn_rows<DT, DP>(k0, kb * 32, q, at), x = attn_rows<DT, DP>(v0, kb * 32, w, at);
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(p[r] - lost, g.scale_log2, -ls));
                    x[r] = t * BN + kb * 32 + 4 * half + 8 * (r / 4) + r % 4 < lim ? e * (x[r] - es) : 0.0f;
                }
                attn_cols<DT, DP>(dq, k0, kb * 32, x, at);
            }
        }
        t1 = t0;
    }
    auto step = [&](int t, const S *kt, const S *vt) {
        at.fresh();
        const int key0 = t * BN + 4 * half;
        const bool mask = (t + 1) * BN > lim_first;
#pragma unroll
        for (int kb = 0; kb < NKB; kb++) {
            auto nothing = [](auto, auto) {};
            floatx16 p, x;
            attn_rows_beside<DT, DP, 2>(p, kt, kb * 32, [&](int f) { return q[f]; }, at, nothing);
            attn_rows_beside<DT, DP, 2>(x, vt, kb * 32, [&](int f) { return w[f]; }, at, [&](auto U, auto N) {
                attn_share(U, N, [&](int r) {
                    float y = __builtin_amdgcn_exp2f(fmaf(p[r], g.scale_log2, -ls));
                    asm volatile("" : "+v"(y));  // here, beside the products
                    p[r] = y;
                });
            });
            if (mask) {
#pragma unroll
                for (int r = 0; r < 16; r++) p[r] = key0 + kb * 32 + 8 * (r / 4) + r % 4 < lim ? p[r] : 0.0f;
            }
#pragma unroll
            for (int r = 0; r < 16; r++) x[r] = p[r] * (x[r] - es);
            attn_cols_beside<DT, DP, 2>(dq, kt, kb * 32, x, at, nothing);
        }
    };
    auto load = [&](int t, S *kt, S *vt) {
        kl.load(ks, g.size, t * BN, kt, wave, lane);
        vl.load(vs, g.size, t * BN, vt, wave, lane);
    };
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
    if (!live) return;
    const long long to = b * g.o_bs + (sq.row + qi) * g.o_ts + hq * g.o_hs;
#pragma unroll
    for (int d = 0; d < ND; d++) {
        auto value = [&](int r) { return dq[d][r] * g.scale; };
        if (g.splits > 1) attn_store_block<PT_FLOAT32>(g.part_o + blockIdx.y * g.part_step + to, d * 32, g.size, half, value);
        else attn_store_block<DT>((S *)g.dq + to, d * 32, g.size, half, value);
    }
}

// ------------------------------------------------------------- launches
// Of one element type (pt_attention_{bf16,f16,f32}.hip).  `vec`: every row
// of every operand starts on 16 bytes and its size fills whole chunks.
template <int DT> void launch_attention(const AttnArgs &g, bool token, bool vec, unsigned blocks, hipStream_t s);
template <int DT> void launch_attention_dkv(const AttnArgs &g, bool vec, unsigned blocks, hipStream_t s);
template <int DT> void launch_attention_dq(const AttnArgs &g, bool vec, unsigned blocks, hipStream_t s);
// streamed rows of a step of the gradient kernels
template <int DT> int attention_backward_tile(int size);

}  // namespace pt
