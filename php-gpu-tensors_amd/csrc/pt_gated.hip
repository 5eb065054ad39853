// Gated projection h = act(x gate) * (x up) and its gradients for gfx950:
//   dg = dh u act'(g),  du = dh act(g)   (g, u: the two products)
//   dx = dg gate^T + du up^T,  dgate = x^T dg,  dup = x^T du.
// Forms, by the rows and the type:
//   16 bits, more than 64 rows: products over a pair of matrices in one
//     kernel (pt_gated_ring.hip), bound by the matrix cores.
//   64 rows or fewer (float32: 32, whose matrix instructions are slower):
//     k_gated_few, bound by the weights' bytes: one row of bfloat16 through
//     4096 x 16384 twice 42-48 us (5.6-6.4 TB/s).
//   float32, more rows: the same products in fp32 (pt_gated_wide.hip), and
//     large gradients by the plain fp32 ring product.
#include "pt_gated.h"

#include <algorithm>

namespace pt {

// ------------------------------------------------------------- few rows
// The weights stream once, in place and at any alignment.  A wave owns a
// strip of columns of both matrices (a 16-byte pack in each of 16 lanes: 128
// columns in 16 bits, 64 in 32) and takes steps of 32 k: lane l loads 8 rows,
// k = 8 (l / 16) .. + 7, of both.  16 bits: those are an 8 x 8 block, whose
// columns, brought side by side by byte permutations (half an instruction
// per element), are the B operands of 8 16x16x32 MFMAs, the c-th of which
// yields each lane's column c; x, 16 rows of it, is the A operand as it
// lies.  32 bits: each loaded row is the B operand of 4 16x16x4 MFMAs.  So no
// weight passes through LDS.  One matrix's loads of the next step go into
// the registers that its products have just left, while the other's are
// multiplied.  The k-steps go to the 8 waves of a block and to S blocks in
// turn; the waves' sums meet in LDS, where each wave adds an eighth of the
// columns in order, and the blocks' in a second kernel.
constexpr int kFewWaves = 8;
constexpr int kFewRows16 = 64, kFewRows32 = 32;  // the most rows
typedef unsigned gd_u32x4 __attribute__((ext_vector_type(4), aligned(1)));

template <int DT, int MT, int NC>
__global__ __launch_bounds__(64 * kFewWaves) void k_gated_few(PairArgs g)
{
    using S = typename GE<DT>::S;
    constexpr int XV = 16 / sizeof(S);  // elements of x in 16 bytes
    typedef unsigned words __attribute__((ext_vector_type(NC * sizeof(S) / 4), aligned(1)));
    constexpr int NW = NC * sizeof(S) / 4;
    constexpr bool LOW = DT != PT_FLOAT32;
    constexpr int SUMS = 2 * NC * 4;    // of a lane and 16 rows
    __shared__ float box[kFewWaves][SUMS][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kg = lane >> 4, n0 = blockIdx.x * 16 * NC + (lane & 15) * NC, at = min(n0, g.N - NC);
    const S *B[2] = {(const S *)g.b0 + at, (const S *)g.b1 + at};
    const S *x[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) x[m] = (const S *)g.a0 + (long long)min(m * 16 + (lane & 15), g.M - 1) * g.lda;

    floatx4 acc[MT][2][NC];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int c = 0; c < NC; c++) acc[m][j][c] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

    words w[2][8];
    gd_u32x4 xv[MT][LOW ? 1 : 2];
    // rows past K: the last one again, taken as zeros below
    auto load_w = [&](auto J, int k0) {
        constexpr int j = decltype(J)::value;
        const int k = k0 + kg * 8;
        if (k0 + 32 <= g.K) {  // uniform
            const S *p = B[j] + (long long)k * g.ldb;
#pragma unroll
            for (int i = 0; i < 8; i++) w[j][i] = __builtin_nontemporal_load((const words *)(p + (long long)i * g.ldb));
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) w[j][i] = *(const words *)(B[j] + (long long)min(k + i, g.K - 1) * g.ldb);
        }
    };
    auto load_x = [&](int k0) {
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int q = 0; q < (LOW ? 1 : 2); q++) {
                const int kx = k0 + kg * 8 + q * XV;
                if (k0 + 32 <= g.K) xv[m][q] = *(const gd_u32x4 *)(x[m] + kx);  // uniform
                else {
                    union { gd_u32x4 raw; S s[XV]; } u;
#pragma unroll
                    for (int c = 0; c < XV; c++) u.s[c] = kx + c < g.K ? x[m][kx + c] : (S)0;
                    xv[m][q] = u.raw;
                }
            }
    };
    auto multiply = [&](auto J, int k0) {
        constexpr int j = decltype(J)::value;
        if (k0 + 32 > g.K) {  // uniform: what the last step has past K is zeros
            const int k = k0 + kg * 8;
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int d = 0; d < NW; d++) w[j][i][d] = k + i < g.K ? w[j][i][d] : 0u;
        }
        if constexpr (LOW) {
            using Frag = typename FragT<DT>::type;
#pragma unroll
            for (int d = 0; d < NW; d++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    gd_u32x4 col;
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        col[i] = __builtin_amdgcn_perm(w[j][2 * i + 1][d], w[j][2 * i][d], h ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        floatx4 &to = acc[m][j][2 * d + h];
                        const Frag fx = __builtin_bit_cast(Frag, xv[m][0]), fw = __builtin_bit_cast(Frag, col);
                        if constexpr (DT == PT_BFLOAT16) to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fx, fw, to, 0, 0, 0);
                        else to = __builtin_amdgcn_mfma_f32_16x16x32_f16(fx, fw, to, 0, 0, 0);
                    }
                }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int c = 0; c < NC; c++)
                        acc[m][j][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(xv[m][i / 4][i % 4]),
                                                                            __uint_as_float(w[j][i][c]), acc[m][j][c], 0, 0, 0);
        }
    };
    const int step = 32 * kFewWaves * g.split;
    int k0 = 32 * ((int)blockIdx.y * kFewWaves + wave);
    if (k0 < g.K) {
        load_w(IC<0>{}, k0);
        load_x(k0);
        load_w(IC<1>{}, k0);
        for (;;) {
            const int next = k0 + step;
            multiply(IC<0>{}, k0);
            if (next < g.K) load_w(IC<0>{}, next);
            multiply(IC<1>{}, k0);
            if (next >= g.K) break;
            load_x(next);
            load_w(IC<1>{}, next);
            k0 = next;
        }
    }
    // Each wave adds an eighth of the sums over the waves, in their order, and
    // stores: SUMS / 8 of them are 4 rows of one column (two in 16 bits) of
    // the first product or of the second, so waves w and w + 4 hold the same
    // columns of the two and meet once more.
    constexpr int MINE = SUMS / kFewWaves;
    const long long plane = (long long)g.M * g.n_out;
    const int live = n0 < g.n_out ? min(NC, g.n_out - at) : 0;
#pragma unroll
    for (int m = 0; m < MT; m++) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) box[wave][(j * NC + c) * 4 + e][lane] = acc[m][j][c][e];
        __syncthreads();
        float sum[MINE];
#pragma unroll
        for (int i = 0; i < MINE; i++) {
            sum[i] = box[0][wave * MINE + i][lane];
#pragma unroll
            for (int v = 1; v < kFewWaves; v++) sum[i] += box[v][wave * MINE + i][lane];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MINE; i++) box[0][wave * MINE + i][lane] = sum[i];
        __syncthreads();
        // lane: rows 4 (l / 16) + e, columns at .. at + NC - 1.  The lane
        // whose pack was moved back from the end stores what its neighbour
        // stores too.
#pragma unroll
        for (int i = 0; i < MINE / 2; i++) {
            const int q = wave * (MINE / 2) + i, c = q / 4, e = q % 4, row = m * 16 + kg * 4 + e;
            if (row >= g.M || c >= live) continue;
            const float p = box[0][q][lane], u = box[0][NC * 4 + q][lane];
            const long long to = (long long)row * g.n_out + at + c;
            if (g.split > 1) {
                float *part = g.parts + (long long)blockIdx.y * 2 * plane + to;
                part[0] = p;
                part[plane] = u;
                continue;
            }
            if (g.c1) gated_keep<DT>(g.c1, plane, to, p, u);
            store_c<DT>(g.c0, (size_t)to, gated_act<LOW>(g.act, p) * u);
        }
    }
}

// ------------------------------------------------- passes over elements
// V elements from p at any element boundary
template <int DT, int V>
__device__ __forceinline__ void gd_load(const typename GE<DT>::S *p, int live, float (&v)[V])
{
    using S = typename GE<DT>::S;
    if (live >= V) {
#pragma unroll
        for (int q = 0; q < V / GE<DT>::PK; q++) {
            union { gd_u32x4 raw; S s[GE<DT>::PK]; } u;
            u.raw = *(const gd_u32x4 *)(p + q * GE<DT>::PK);
#pragma unroll
            for (int k = 0; k < GE<DT>::PK; k++) v[q * GE<DT>::PK + k] = DType<DT>::to_c(u.s[k]);
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < V; k++) v[k] = k < live ? DType<DT>::to_c(p[k]) : 0.0f;
}

// 8 elements of a product as the gradient keeps it in 24 bits
__device__ __forceinline__ void gd_load_kept(const void *kept, long long n, int product, long long i, int live, float (&v)[8])
{
    const uint16_t *high = (const uint16_t *)((const char *)kept + kept_plane(n, product, false)) + i;
    const uint8_t *low = (const uint8_t *)kept + kept_plane(n, product, true) + i;
    typedef unsigned u32x2 __attribute__((ext_vector_type(2), aligned(1)));
    if (live >= 8) {
        const gd_u32x4 h = __builtin_nontemporal_load((const gd_u32x4 *)high);
        const u32x2 l = __builtin_nontemporal_load((const u32x2 *)low);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = kept_value(h[k / 2] >> (k & 1 ? 16 : 0) & 0xffffu, l[k / 4] >> (8 * (k % 4)) & 0xffu);
        return;
    }
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = k < live ? kept_value(high[k], low[k]) : 0.0f;
}

// Two fp32 matrices [rows][cols] side by side, or (BACK) apart again, in packs
// of 4.
template <bool BACK>
__global__ __launch_bounds__(256) void k_gated_beside(float *a, float *b, float *both, int rows, int cols)
{
    typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
    const int packs = cols / 4;
    const long long n = (long long)rows * packs;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const long long row = i / packs, at = row * 2 * cols + (i - row * packs) * 4;
        float4u *p = (float4u *)a + i, *q = (float4u *)b + i, *r = (float4u *)(both + at), *t = (float4u *)(both + at + cols);
        if constexpr (BACK) {
            *p = *r;
            *q = *t;
        } else {
            *r = *p;
            *t = *q;
        }
    }
}

// Matrices (blockIdx.y) of 16-bit elements into rows of `pitch`, zeros past
// the end; one launch for all that a call copies (5 us less where x and the
// weights are both copied).  1000 x 2731 twice from HBM: 9 us.
struct PackJob {
    const uint16_t *from;
    uint16_t *to;
    int rows, cols, pitch;
};
struct PackArgs {
    PackJob job[3];
};
__global__ __launch_bounds__(256) void k_gated_pack(PackArgs a)
{
    const PackJob &j = a.job[blockIdx.y];
    const int packs = j.pitch / 8;
    const long long total = (long long)j.rows * packs;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long row = i / packs;
        const int c = (int)(i - row * packs) * 8, live = j.cols - c;
        const uint16_t *from = j.from + row * j.cols + c;
        union { gd_u32x4 raw; uint16_t s[8]; } u;
        if (live >= 8) u.raw = *(const gd_u32x4 *)from;
        else
#pragma unroll
            for (int k = 0; k < 8; k++) u.s[k] = k < live ? from[k] : (uint16_t)0;
        *(gd_u32x4 *)(j.to + row * j.pitch + c) = u.raw;
    }
}

// The transpose of rows x cols 16-bit elements, in rows of `pitch` (a
// multiple of 8, zeros past `rows`): a 64 x 64 tile through LDS.
__device__ __forceinline__ void gated_transpose(const uint16_t *from, uint16_t *to, int rows, int cols, int pitch, int r0, int c0,
                                                uint16_t (&tile)[64][66])
{
    const int a = threadIdx.x & 7, b = threadIdx.x >> 3;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int r = r0 + b + 32 * h, c = c0 + a * 8;
        union { gd_u32x4 raw; uint16_t s[8]; } u;
        if (r < rows && c + 8 <= cols) u.raw = *(const gd_u32x4 *)(from + (long long)r * cols + c);
        else
#pragma unroll
            for (int k = 0; k < 8; k++) u.s[k] = r < rows && c + k < cols ? from[(long long)r * cols + c + k] : (uint16_t)0;
#pragma unroll
        for (int k = 0; k < 8; k++) tile[a * 8 + k][b + 32 * h] = u.s[k];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int c = c0 + b + 32 * h, r = r0 + a * 8;
        if (c >= cols || r >= pitch) continue;  // (pitch and r are multiples of 8)
        union { gd_u32x4 raw; uint16_t s[8]; } u;
#pragma unroll
        for (int k = 0; k < 8; k++) u.s[k] = tile[b + 32 * h][a * 8 + k];
        *(gd_u32x4 *)(to + (long long)c * pitch + r) = u.raw;
    }
}

// dg and du of 8 elements from `from` on, `live` of them, from the upstream
// gradient and both products; the others are zeros.
template <int DT, int GDT>
__device__ __forceinline__ void gd_slopes(const void *kept, const void *grad, int act, long long plane, long long from, int live,
                                          float (&dg)[8], float (&du)[8])
{
    using S = typename GE<DT>::S;
    float g[8], u[8], dh[8];
    if constexpr (DT == PT_FLOAT32) {
        gd_load<DT, 8>((const S *)kept + from, live, g);
        gd_load<DT, 8>((const S *)kept + plane + from, live, u);
    } else {
        gd_load_kept(kept, plane, 0, from, live, g);
        gd_load_kept(kept, plane, 1, from, live, u);
    }
    gd_load<GDT, 8>((const typename GE<GDT>::S *)grad + from, live, dh);
#pragma unroll
    for (int k = 0; k < 8; k++) {
        float value, slope;
        gated_slope<DT != PT_FLOAT32>(act, g[k], value, slope);
        dg[k] = k < live ? dh[k] * u[k] * slope : 0.0f;
        du[k] = k < live ? dh[k] * value : 0.0f;
    }
}

// dg and du into rows `pitch` elements apart from d and d + second on, zeros
// in columns `cols` to `padded` - 1.  A thread takes 8 columns.  Blocks from
// `slopes` on transpose x beside it, one 64 x 64 tile each, in one launch
// less.  HBM-bound: 8192 x 8192 in bfloat16 with a transpose of 8192 x 2048
// 160-170 us, 5.3 TB/s.  float16: twice, multiplied by the rows' powers of
// two into d and by the columns' into e (either may be null): 200 us.
struct SlopeArgs {
    const void *kept, *grad;
    void *d;
    long long second;
    int rows, cols, padded, pitch, act;
    unsigned slopes;         // blocks
    const uint16_t *x;       // [rows][inner]
    uint16_t *xt;            // [inner][across]
    int inner, across;
    void *e;
    const int8_t *row_shift, *column_shift;  // [rows], [2][cols] and 8 bytes more
};
template <int DT, int GDT>
__global__ __launch_bounds__(256) void k_gated_slope(SlopeArgs a)
{
    using S = typename GE<DT>::S;
    __shared__ uint16_t tile[64][66];
    if (blockIdx.x >= a.slopes) {
        const int t = (int)(blockIdx.x - a.slopes), wide = (a.inner + 63) / 64;
        gated_transpose(a.x, a.xt, a.rows, a.inner, a.across, t / wide * 64, t % wide * 64, tile);
        return;
    }
    const int packs = (a.cols + 7) / 8;
    const long long total = (long long)a.rows * packs, plane = (long long)a.rows * a.cols;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)a.slopes * 256) {
        const long long row = i / packs;
        const int c = (int)(i - row * packs) * 8, live = min(8, a.cols - c), room = min(8, a.padded - c);
        float dg[8], du[8];
        gd_slopes<DT, GDT>(a.kept, a.grad, a.act, plane, row * a.cols + c, live, dg, du);
        auto store = [&](void *d, const float (&p)[8], const float (&q)[8]) {
            S v[8], w[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                v[k] = DType<DT>::from_c(p[k]);
                w[k] = DType<DT>::from_c(q[k]);
            }
            S *to = (S *)d + row * a.pitch + c;
            if (room == 8) {
#pragma unroll
                for (int k = 0; k < 8; k += GE<DT>::PK) {
                    *(gd_u32x4 *)(to + k) = *(gd_u32x4 *)(v + k);
                    *(gd_u32x4 *)(to + a.second + k) = *(gd_u32x4 *)(w + k);
                }
            } else {
                for (int k = 0; k < room; k++) {
                    to[k] = v[k];
                    to[a.second + k] = w[k];
                }
            }
        };
        if constexpr (DT == PT_FLOAT16) {
            float p[8], q[8];
            if (a.d) {
                const int shift = a.row_shift[row];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    p[k] = ldexpf(dg[k], shift);
                    q[k] = ldexpf(du[k], shift);
                }
                store(a.d, p, q);
            }
            if (a.e) {
                // (past the last column: another shift of a zero)
                typedef int8_t shifts __attribute__((ext_vector_type(8), aligned(1)));
                const shifts x = *(const shifts *)(a.column_shift + c), y = *(const shifts *)(a.column_shift + a.cols + c);
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    p[k] = ldexpf(dg[k], x[k]);
                    q[k] = ldexpf(du[k], y[k]);
                }
                store(a.e, p, q);
            }
        } else {
            store(a.d, dg, du);
        }
    }
}

// the largest over the 2^log2 lanes that share a row (log2 is uniform), by DPP up to 16
__device__ __forceinline__ float gd_top(float v, int log2)
{
    auto with = [](float x, auto CTRL) {
        return fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(CTRL)::value, 0xF, 0xF, false)));
    };
    if (log2 == 6) return wave_all(v, FMax{});
    if (log2 > 0) v = with(v, IC<0xB1>{});
    if (log2 > 1) v = with(v, IC<0x4E>{});
    if (log2 > 2) v = with(v, IC<0x141>{});
    if (log2 > 3) v = with(v, IC<0x140>{});
    if (log2 > 4) v = fmaxf(v, __shfl_xor(v, 16, PT_WAVE));
    return v;
}

// float16: the largest finite |dg| and |du| of each row and of each column (the
// two apart), of the rows' and columns' parts that a block takes; the second
// kernel takes the largest over the parts, in any order the same.  A wave walks
// `steps` rows, 512 columns of each (fewer columns: as many rows at once as
// fill it), so a row is reduced over its lanes and a column stays in one.
// 8192 x 8192: 119-124 us (4.4 TB/s) and 5.
struct RangeArgs {
    const void *kept, *grad;
    int rows, cols, act;
    int lanes_log2, steps;   // lanes of a row; a wave's steps
    float *row_part;         // [gridDim.x][rows], or null
    float *column_part;      // [gridDim.y][2][cols], or null
};
template <int GDT>
__global__ __launch_bounds__(256) void k_gated_range(RangeArgs a)
{
    __shared__ float box[4][16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lanes = 1 << a.lanes_log2, at_once = 64 >> a.lanes_log2;
    const int c = (blockIdx.x * lanes + (lane & (lanes - 1))) * 8, live = max(0, min(8, a.cols - c));
    const long long plane = (long long)a.rows * a.cols;
    const long long r0 = ((long long)blockIdx.y * 4 + wave) * a.steps * at_once + (lane >> a.lanes_log2);
    float top[16];
#pragma unroll
    for (int k = 0; k < 16; k++) top[k] = 0.0f;
#pragma unroll 4
    for (int s = 0; s < a.steps; s++) {
        const long long row = r0 + (long long)s * at_once;
        const int n = row < a.rows ? live : 0;
        float dg[8], du[8], most = 0.0f;
        gd_slopes<PT_FLOAT16, GDT>(a.kept, a.grad, a.act, plane, n ? row * a.cols + c : 0, n, dg, du);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float p = fabsf(dg[k]), q = fabsf(du[k]);
            top[k] = fmaxf(top[k], p < INFINITY ? p : 0.0f);
            top[8 + k] = fmaxf(top[8 + k], q < INFINITY ? q : 0.0f);
            most = fmaxf(most, fmaxf(p < INFINITY ? p : 0.0f, q < INFINITY ? q : 0.0f));
        }
        most = gd_top(most, a.lanes_log2);
        if (a.row_part && !(lane & (lanes - 1)) && row < a.rows) a.row_part[(long long)blockIdx.x * a.rows + row] = most;
    }
    if (!a.column_part) return;  // uniform
#pragma unroll
    for (int k = 0; k < 16; k++) {
        for (int m = lanes; m < 64; m <<= 1) top[k] = fmaxf(top[k], __shfl_xor(top[k], m, PT_WAVE));
        box[wave][k][lane] = top[k];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * lanes; i += 256) {
        const int j = i / (8 * lanes), at = i - j * 8 * lanes, column = blockIdx.x * lanes * 8 + at, k = j * 8 + at % 8;
        if (column >= a.cols) continue;
        float t = box[0][k][at / 8];
        for (int w = 1; w < 4; w++) t = fmaxf(t, box[w][k][at / 8]);
        a.column_part[((long long)blockIdx.y * 2 + j) * a.cols + column] = t;
    }
}

// The powers of two from the parts' largest values: items 0 to rows - 1 are
// rows, the 2 cols behind them columns; a block takes 64, each of its waves
// every 16th part.
struct ShiftArgs {
    const float *row_part, *column_part;
    int rows, columns;   // 0: none wanted
    int row_parts, column_parts;
    int8_t *shift;       // [rows + columns]
};
constexpr int kShiftWaves = 16;
__global__ __launch_bounds__(64 * kShiftWaves) void k_gated_shift(ShiftArgs a)
{
    __shared__ float box[kShiftWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long items = (long long)a.rows + a.columns, i = (long long)blockIdx.x * 64 + lane;
    const bool row = i < a.rows;
    const float *from = row ? a.row_part + i : a.column_part + (i - a.rows);
    const int parts = i < items ? (row ? a.row_parts : a.column_parts) : 0, step = row ? a.rows : a.columns;
    float top = 0.0f;
#pragma unroll 8
    for (int k = wave; k < parts; k += kShiftWaves) top = fmaxf(top, from[(long long)k * step]);
    box[wave][lane] = top;
    __syncthreads();
    if (wave || i >= items) return;
#pragma unroll
    for (int w = 1; w < kShiftWaves; w++) top = fmaxf(top, box[w][lane]);
    a.shift[i] = (int8_t)gated_shift(top);
}

// ------------------------------------------------------------- the calls
static int round8(int n) { return (n + 7) / 8 * 8; }
static unsigned grid_for(long long items) { return (unsigned)std::min<long long>((items + 255) / 256, 1 << 20); }

// Scratch of one call, given back in the stream's order.
struct GatedScratch {
    hipStream_t s;
    void *held[10];
    int count = 0;
    explicit GatedScratch(hipStream_t stream) : s(stream) {}
    ~GatedScratch()
    {
        while (count) scratch_free(held[--count], s);
    }
    pt_status take(void **p, size_t bytes)
    {
        PT_TRY(scratch_alloc(p, bytes, s));
        held[count++] = *p;
        return PT_OK;
    }
    // A 16-bit matrix whose rows start at 16-byte boundaries: itself, or a copy
    // that pack() makes.
    PackArgs packs;
    int jobs = 0;
    pt_status rows16(const void *a, int rows, int cols, const void **to, bool copy)
    {
        *to = a;
        if (!copy) return PT_OK;
        uint16_t *p = nullptr;
        PT_TRY(take((void **)&p, (size_t)rows * round8(cols) * 2));
        packs.job[jobs++] = {(const uint16_t *)a, p, rows, cols, round8(cols)};
        *to = p;
        return PT_OK;
    }
    void pack()
    {
        long long most = 0;
        for (int i = 0; i < jobs; i++) most = std::max(most, (long long)packs.job[i].rows * (packs.job[i].pitch / 8));
        if (jobs) k_gated_pack<<<dim3(grid_for(most), jobs), 256, 0, s>>>(packs);
        jobs = 0;
    }
    // both weights alike, at one pitch
    pt_status weights16(const void *gate, const void *up, int rows, int cols, PairArgs &g)
    {
        const bool copy = cols % 8 || (((uintptr_t)gate | (uintptr_t)up) & 15);
        PT_TRY(rows16(gate, rows, cols, &g.b0, copy));
        PT_TRY(rows16(up, rows, cols, &g.b1, copy));
        g.ldb = round8(cols);
        return PT_OK;
    }
};

static pt_status gated_check(const pt_gated_desc *d)
{
    if (!d) return fail(PT_ERR_INVALID, "gated projection description missing");
    if (d->dtype != PT_FLOAT32 && d->dtype != PT_FLOAT16 && d->dtype != PT_BFLOAT16)
        return fail(PT_ERR_INVALID, "gated projection takes float32, float16 or bfloat16");
    if (d->activation < PT_GATE_SILU || d->activation > PT_GATE_SIGMOID)
        return fail(PT_ERR_INVALID, "gated projection activation %d is not known", d->activation);
    if (d->rows < 0 || d->inner < 0 || d->outer < 0) return fail(PT_ERR_INVALID, "gated projection sizes must not be negative");
    if (d->rows > kPairPitch || d->inner > kPairPitch || d->outer > kPairPitch)
        return fail(PT_ERR_UNSUPPORTED, "gated projection takes at most %lld rows, and elements in each", kPairPitch);
    return PT_OK;
}

static pt_status zeros(void *p, int dtype, size_t n, pt_stream_t stream)
{
    const pt_scalar_t zero = {{0.0}, dtype};
    return p && n ? pt_fill(p, dtype, n, &zero, stream) : PT_OK;
}

// C = A B, fp32, strides in elements
static pt_status product_f32(const float *a, size_t am, size_t ak, const float *b, size_t bk, size_t bn, float *c, int m, int n,
                             int k, pt_stream_t stream)
{
    const int sa[2] = {m, k}, sb[2] = {k, n}, sc[2] = {m, n};
    const size_t ta[2] = {am, ak}, tb[2] = {bk, bn};
    return pt_matmul(a, b, c, PT_FLOAT32, sa, ta, 2, sb, tb, 2, sc, 2, stream);
}

// A product over a pair of matrices in fp32
static pt_status run_wide(PairArgs &g, int form, int store, GatedScratch &scratch)
{
    int tm;
    wide_plan(g, form, tm);
    if (g.split > 1) PT_TRY(scratch.take((void **)&g.parts, (size_t)g.split * (form == WIDE_SUM ? 1 : 2) * g.M * g.n_out * sizeof(float)));
    launch_wide(g, tm, form, store, scratch.s);
    return PT_OK;
}

// Wide strips, whose k-steps are split over up to a block for every CU; strips
// of 8-byte packs, without a split, where the split's second kernel (4.5 us)
// costs more than the CUs that they leave idle: a CU streams 33 GB/s, all of
// them 5.3 TB/s.  One row of bfloat16, wide against narrow: 4096 x 16384 54
// and 49 us, 512 x 2048 8.5 and 5.3, 4096 x 4096 19 and 35.
template <int DT>
static pt_status launch_few(PairArgs &g, GatedScratch &scratch, hipStream_t s)
{
    constexpr int NC = GE<DT>::PK;
    constexpr bool LOW = DT != PT_FLOAT32;
    // (16 bits, more than 32 rows: the sums of a wide strip leave no registers)
    const int wide = (g.n_out + 16 * NC - 1) / (16 * NC), narrow = (g.n_out + 8 * NC - 1) / (8 * NC), steps = (g.K + 31) / 32;
    const bool must = LOW && g.M > 32;
    const double bytes = 2.0 * g.K * g.n_out * sizeof(typename GE<DT>::S);
    g.split = std::max(1, std::min({256 / (must ? narrow : wide), steps / kFewWaves, 16}));
    const bool alone = g.split > 1 && bytes / (std::min(narrow, 160) * 33e9) < bytes / 5.3e12 + 4.5e-6, thin = must || alone;
    if (alone) g.split = 1;
    if (g.split > 1) PT_TRY(scratch.take((void **)&g.parts, (size_t)g.split * 2 * g.M * g.n_out * sizeof(float)));
    const dim3 grid(thin ? narrow : wide, g.split);
    auto go = [&](auto NCC) {
        constexpr int N = decltype(NCC)::value;
        if (g.M <= 16) k_gated_few<DT, 1, N><<<grid, 64 * kFewWaves, 0, s>>>(g);
        else if (!LOW || N == NC || g.M <= 32) k_gated_few<DT, 2, N><<<grid, 64 * kFewWaves, 0, s>>>(g);
        else if constexpr (LOW && N < NC) k_gated_few<DT, 4, N><<<grid, 64 * kFewWaves, 0, s>>>(g);
    };
    if (thin) go(IC<NC / 2>{});
    else go(IC<NC>{});
    if (g.split > 1) launch_pair_join(g, DT, false, g.c1 ? GATED_KEPT : GATED_PRODUCT, s);
    return PT_OK;
}

static pt_status gated_run(const pt_gated_desc *d, const void *x, const void *gate, const void *up, void *h, void *kept,
                           pt_stream_t stream)
{
    hipStream_t s = stream_of(stream);
    GatedScratch scratch(s);
    const int M = d->rows, K = d->inner, F = d->outer;
    const size_t size = dtype_size(d->dtype), n = (size_t)M * F;
    PairArgs g = {};
    g.M = M;
    g.act = d->activation;
    g.n_out = F;
    g.c0 = h;
    g.c1 = kept;
    g.a0 = x;
    g.b0 = gate;
    g.b1 = up;
    g.lda = K;
    g.ldb = g.N = F;
    g.K = g.kb = K;
    const int pack = (int)(16 / size);
    if (M <= (d->dtype == PT_FLOAT32 ? kFewRows32 : kFewRows16) && F >= pack) {
        if (d->dtype == PT_FLOAT32) return launch_few<PT_FLOAT32>(g, scratch, s);
        return d->dtype == PT_FLOAT16 ? launch_few<PT_FLOAT16>(g, scratch, s) : launch_few<PT_BFLOAT16>(g, scratch, s);
    }
    if (d->dtype == PT_FLOAT32) return run_wide(g, WIDE_COLUMNS, kept ? GATED_KEPT : GATED_PRODUCT, scratch);
    PT_TRY(scratch.rows16(x, M, K, &g.a0, K % 8 || ((uintptr_t)x & 15)));
    PT_TRY(scratch.weights16(gate, up, K, F, g));
    scratch.pack();
    g.lda = round8(K);
    // (of K rounded to 8, A's elements past K are zeros or B's rows past it are out of range)
    g.K = round8(K);
    g.N = (int)g.ldb;
    int tm;
    pair_plan(g, true, tm);
    if (g.split > 1) PT_TRY(scratch.take((void **)&g.parts, (size_t)g.split * 2 * n * sizeof(float)));
    launch_pair_columns(g, d->dtype, tm, kept ? GATED_KEPT : GATED_PRODUCT, s);
    return PT_OK;
}

// Large products of whole packs and of 512 rows or more: the plain ring
// product, whose loads go to LDS by themselves, holds 95-100 % of the matrix
// cores at its clock where the pair kernel holds 80, which pays for copies of
// the weights, and of their gradients, side by side: both ways 8192 x 1024 x
// 1024 801 us, 934 with the pair kernel, 4096 x 784 x 1024 383 and 415; but 1000 x 768 x
// 2048 223 and 216, and of 4096 x 14336 64 rows 893 and 529, 256 1741 and 1588,
// 512 2958 and 2996.
static bool gated_ring_f32(int M, int K, int F) { return K % 4 == 0 && F % 4 == 0 && M >= 512 && (double)M * K * F > 2.5e9; }

static pt_status gated_backward_f32(const pt_gated_desc *d, const float *x, const float *gate, const float *up, const void *kept,
                                    const void *grad, float *dx, float *dgate, float *dup, GatedScratch &scratch, pt_stream_t stream)
{
    hipStream_t s = scratch.s;
    const int M = d->rows, K = d->inner, F = d->outer;
    const bool ring = gated_ring_f32(M, K, F);
    // dg and du side by side, where one product takes both contractions of dx
    const long long pitch = ring ? 2 * F : F, second = ring ? F : ((long long)M * F + 3) / 4 * 4;
    float *dg = nullptr, *both = nullptr;
    PT_TRY(scratch.take((void **)&dg, 2 * (ring ? (size_t)M * F : (size_t)second) * sizeof(float)));
    SlopeArgs a = {};
    a.kept = kept;
    a.grad = grad;
    a.d = dg;
    a.second = second;
    a.rows = M;
    a.cols = a.padded = F;
    a.pitch = (int)pitch;
    a.act = d->activation;
    a.slopes = grid_for((long long)M * ((F + 7) / 8));
    k_gated_slope<PT_FLOAT32, PT_FLOAT32><<<a.slopes, 256, 0, s>>>(a);
    const unsigned blocks = grid_for((long long)K * F / 4);
    if (ring) PT_TRY(scratch.take((void **)&both, (size_t)K * 2 * F * sizeof(float)));
    if (dx && ring) {
        k_gated_beside<false><<<blocks, 256, 0, s>>>((float *)gate, (float *)up, both, K, F);
        PT_TRY(product_f32(dg, pitch, 1, both, 1, pitch, dx, M, K, 2 * F, stream));
    } else if (dx) {
        PairArgs g = {};
        g.a0 = dg;
        g.a1 = dg + second;
        g.b0 = gate;
        g.b1 = up;
        g.lda = g.ldb = g.K = F;
        g.M = M;
        g.N = g.n_out = K;
        g.c0 = dx;
        PT_TRY(run_wide(g, WIDE_SUM, GATED_PRODUCT, scratch));
    }
    if (dgate && ring) {
        PT_TRY(product_f32(x, 1, K, dg, pitch, 1, both, K, 2 * F, M, stream));
        k_gated_beside<true><<<blocks, 256, 0, s>>>(dgate, dup, both, K, F);
    } else if (dgate) {
        PairArgs g = {};
        g.a0 = x;
        g.b0 = dg;
        g.b1 = dg + second;
        g.lda = g.M = K;
        g.ldb = g.N = g.n_out = F;
        g.K = M;
        g.c1 = dgate;
        g.c2 = dup;
        PT_TRY(run_wide(g, WIDE_TURNED, GATED_BOTH, scratch));
    }
    return PT_OK;
}

// The powers of two of float16 gradients, for dx and for the weights' where
// wanted.  A wave walks as many rows as leave 2048 blocks, 16 at most, but so
// many that a column has no more than 256 parts.
static pt_status gated_shifts(SlopeArgs &s, int grad_dtype, bool rows, bool columns, GatedScratch &scratch)
{
    RangeArgs a = {};
    a.kept = s.kept;
    a.grad = s.grad;
    a.rows = s.rows;
    a.cols = s.cols;
    a.act = s.act;
    const int packs = (s.cols + 7) / 8;
    while (a.lanes_log2 < 6 && 1 << a.lanes_log2 < packs) a.lanes_log2++;
    const int at_once = 4 * (64 >> a.lanes_log2), chunks = (packs + (1 << a.lanes_log2) - 1) >> a.lanes_log2;
    const int turns = (s.rows + at_once - 1) / at_once;
    a.steps = (int)std::max<long long>((turns + 255) / 256, std::min<long long>((long long)turns * chunks / 2048, 16));
    const int blocks = (turns + a.steps - 1) / a.steps;
    int8_t *shift = nullptr;
    const size_t many = (rows ? (size_t)s.rows : 0) + (columns ? 2 * (size_t)s.cols : 0);
    PT_TRY(scratch.take((void **)&shift, many + 8));
    const size_t row_parts = rows ? (size_t)chunks * s.rows : 0, column_parts = columns ? (size_t)blocks * 2 * s.cols : 0;
    float *parts = nullptr;
    PT_TRY(scratch.take((void **)&parts, (row_parts + column_parts) * sizeof(float)));
    if (rows) a.row_part = parts;
    if (columns) a.column_part = parts + row_parts;
    const dim3 grid(chunks, blocks);
    if (grad_dtype == PT_FLOAT16) k_gated_range<PT_FLOAT16><<<grid, 256, 0, scratch.s>>>(a);
    else k_gated_range<PT_FLOAT32><<<grid, 256, 0, scratch.s>>>(a);
    const ShiftArgs t = {a.row_part, a.column_part, rows ? s.rows : 0, columns ? 2 * s.cols : 0, chunks, blocks, shift};
    k_gated_shift<<<(unsigned)((many + 63) / 64), 64 * kShiftWaves, 0, scratch.s>>>(t);
    s.row_shift = shift;
    s.column_shift = shift + t.rows;
    return PT_OK;
}

static pt_status gated_backward_run(const pt_gated_desc *d, const void *x, const void *gate, const void *up, const void *kept,
                                    const void *grad, int grad_dtype, void *dx, void *dgate, void *dup, pt_stream_t stream)
{
    hipStream_t s = stream_of(stream);
    GatedScratch scratch(s);
    const int M = d->rows, K = d->inner, F = d->outer, pitch = round8(F);
    const bool half = d->dtype == PT_FLOAT16;
    if (d->dtype == PT_FLOAT32)
        return gated_backward_f32(d, (const float *)x, (const float *)gate, (const float *)up, kept, grad, (float *)dx,
                                  (float *)dgate, (float *)dup, scratch, stream);
    // dg and du for dx, and for the weights' gradients: the same but in float16
    uint16_t *dg = nullptr, *dw = nullptr;
    const long long second = (long long)M * pitch;
    if (dx || !half) PT_TRY(scratch.take((void **)&dg, (size_t)second * 2 * 2));
    if (dgate && half) PT_TRY(scratch.take((void **)&dw, (size_t)second * 2 * 2));
    SlopeArgs a = {};
    a.kept = kept;
    a.grad = grad;
    a.d = dg;
    a.e = dw;
    a.second = second;
    a.rows = M;
    a.cols = F;
    a.padded = a.pitch = pitch;
    a.act = d->activation;
    a.slopes = grid_for((long long)M * (pitch / 8));
    if (half) PT_TRY(gated_shifts(a, grad_dtype, dx, dgate, scratch));
    else dw = dg;
    unsigned blocks = a.slopes;
    if (dgate) {
        a.x = (const uint16_t *)x;
        a.inner = K;
        a.across = round8(M);
        PT_TRY(scratch.take((void **)&a.xt, (size_t)K * a.across * 2));
        blocks += (unsigned)(((long long)K + 63) / 64 * ((a.across + 63) / 64));
    }
    const bool same = grad_dtype == d->dtype;
    if (d->dtype == PT_BFLOAT16) {
        if (same) k_gated_slope<PT_BFLOAT16, PT_BFLOAT16><<<blocks, 256, 0, s>>>(a);
        else k_gated_slope<PT_BFLOAT16, PT_FLOAT32><<<blocks, 256, 0, s>>>(a);
    } else {
        if (same) k_gated_slope<PT_FLOAT16, PT_FLOAT16><<<blocks, 256, 0, s>>>(a);
        else k_gated_slope<PT_FLOAT16, PT_FLOAT32><<<blocks, 256, 0, s>>>(a);
    }
    int tm;
    if (dx) {
        PairArgs g = {};
        g.a0 = dg;
        g.a1 = dg + second;
        g.lda = pitch;
        PT_TRY(scratch.weights16(gate, up, K, F, g));
        scratch.pack();
        g.M = M;
        g.N = g.n_out = K;
        g.K = pitch;
        g.c0 = dx;
        g.shift = a.row_shift;
        pair_plan(g, false, tm);
        if (g.split > 1) PT_TRY(scratch.take((void **)&g.parts, (size_t)g.split * M * K * sizeof(float)));
        launch_pair_sum(g, d->dtype, tm, s);
    }
    if (dgate) {
        PairArgs g = {};
        g.a0 = a.xt;
        g.lda = g.K = a.across;
        g.kb = M;
        g.b0 = dw;
        g.b1 = dw + second;
        g.ldb = g.N = pitch;
        g.n_out = F;
        g.M = K;
        g.c1 = dgate;
        g.c2 = dup;
        g.shift = a.column_shift;
        pair_plan(g, true, tm);
        if (g.split > 1) PT_TRY(scratch.take((void **)&g.parts, (size_t)g.split * 2 * K * F * sizeof(float)));
        launch_pair_columns(g, d->dtype, tm, GATED_BOTH, s);
    }
    return PT_OK;
}

}  // namespace pt

using namespace pt;

extern "C" {

pt_status pt_gated(const pt_gated_desc *d, const void *x, const void *gate, const void *up, void *h, void *kept,
                   pt_stream_t stream)
{
    PT_TRY(gated_check(d));
    const size_t n = (size_t)d->rows * d->outer;
    if (n && (!h || (d->inner && (!x || !gate || !up)))) return fail(PT_ERR_INVALID, "gated projection misses an operand");
    PT_TRY(ensure_init());
    if (!n) return PT_OK;
    if (!d->inner) {  // empty sums: act(0) 0
        PT_TRY(zeros(kept, PT_UINT8, (d->dtype == PT_FLOAT32 ? 8 : 6) * n, stream));
        return zeros(h, d->dtype, n, stream);
    }
    PT_TRY(gated_run(d, x, gate, up, h, kept, stream));
    return check_hip(hipGetLastError(), "gated projection");
}

pt_status pt_gated_backward(const pt_gated_desc *d, const void *x, const void *gate, const void *up, const void *kept,
                            const void *grad, int grad_dtype, void *dx, void *dgate, void *dup, pt_stream_t stream)
{
    PT_TRY(gated_check(d));
    if (grad_dtype != d->dtype && grad_dtype != PT_FLOAT32)
        return fail(PT_ERR_INVALID, "the gated projection's upstream gradient must be float32 or of its dtype");
    if (!dgate != !dup || (!dx && !dgate)) return fail(PT_ERR_INVALID, "gated projection gradient misses a result");
    const bool some = d->rows && d->inner && d->outer;
    if (some && (!x || !gate || !up || !kept || !grad)) return fail(PT_ERR_INVALID, "gated projection gradient misses an operand");
    PT_TRY(ensure_init());
    if (!some) {  // empty sums
        PT_TRY(zeros(dx, d->dtype, (size_t)d->rows * d->inner, stream));
        PT_TRY(zeros(dgate, d->dtype, (size_t)d->inner * d->outer, stream));
        return zeros(dup, d->dtype, (size_t)d->inner * d->outer, stream);
    }
    PT_TRY(gated_backward_run(d, x, gate, up, kept, grad, grad_dtype, dx, dgate, dup, stream));
    return check_hip(hipGetLastError(), "gated projection gradient");
}

}  // extern "C"
