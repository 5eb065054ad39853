// Gated projection h = act(x gate) * (x up) and its gradients for gfx950:
//   dg = dh u act'(g),  du = dh act(g)   (g, u: the two products)
//   dx = dg gate^T + du up^T,  dgate = x^T dg,  dup = x^T du.
// Forms, by the rows and the type:
//   16 bits, more than 64 rows: products over a pair of matrices in one
//     kernel (pt_gated_ring.hip), bound by the matrix cores.
//   64 rows or fewer (float32: 32, whose matrix instructions are slower):
//     k_gated_few, bound by the weights' bytes: one row of bfloat16 through
//     4096 x 16384 twice 42-48 us (5.6-6.4 TB/s).
//   float32, more rows: the framework's fp32 products (94 % of the matrix
//     cores' rate), one for both weights side by side where that is faster,
//     and a pass over both results; fusing would save that pass, 2 % of the
//     time at 4096 inner elements.
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

// h of fp32 products in rows `pitch` elements apart, the second `second`
// behind the first; a thread takes 4 columns.
__global__ __launch_bounds__(256) void k_gated_product(const float *p, float *h, int rows, int cols, int pitch, long long second,
                                                       int act)
{
    const int packs = (cols + 3) / 4;
    const long long total = (long long)rows * packs;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long row = i / packs;
        const int c = (int)(i - row * packs) * 4, live = min(4, cols - c);
        float g[4], u[4];
        gd_load<PT_FLOAT32, 4>(p + row * pitch + c, live, g);
        gd_load<PT_FLOAT32, 4>(p + row * pitch + second + c, live, u);
        gated_products<false>(act, g, u);
        float *to = h + row * cols + c;
        typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
        if (live == 4) *(float4u *)to = float4u{g[0], g[1], g[2], g[3]};
        else
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (k < live) to[k] = g[k];
    }
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

// Two fp32 matrices [rows][cols] side by side, each in `each` columns (zeros
// past the end, also in rows up to `down`), or (BACK) apart again.
template <bool BACK>
__global__ __launch_bounds__(256) void k_gated_beside(float *a, float *b, float *both, int rows, int cols, int down, int each)
{
    const long long n = (long long)(BACK ? rows : down) * each;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const long long row = i / each, c = i - row * each, at = i + row * each, from = row * cols + c;
        const bool live = row < rows && c < cols;
        if constexpr (BACK) {
            if (live) {
                a[from] = both[at];
                b[from] = both[at + each];
            }
        } else {
            both[at] = live ? a[from] : 0.0f;
            both[at + each] = live ? b[from] : 0.0f;
        }
    }
}

__global__ __launch_bounds__(256) void k_gated_sum(float *a, const float *b, long long n)
{
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) a[i] += b[i];
}

// fp32 rows of `cols` in rows of `pitch`, zeros past the end
__global__ __launch_bounds__(256) void k_gated_pitch(const float *from, float *to, long long rows, int cols, int pitch)
{
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * pitch; i += (long long)gridDim.x * 256) {
        const long long row = i / pitch, c = i - row * pitch;
        to[i] = c < cols ? from[row * cols + c] : 0.0f;
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

// dg and du from the upstream gradient and both products, into rows `pitch`
// elements apart from d and d + second on, zeros in columns `cols` to
// `padded` - 1.  A thread takes 8 columns.  Blocks from `slopes` on transpose
// x beside it, one 64 x 64 tile each, in one launch less.  HBM-bound: 8192 x
// 8192 in bfloat16 with a transpose of 8192 x 2048 160-170 us, 5.3 TB/s.
struct SlopeArgs {
    const void *kept, *grad;
    void *d;
    long long second;
    int rows, cols, padded, pitch, act;
    int kept_pitch;          // float32: both products' rows, and where the second one's begin
    long long kept_second;
    unsigned slopes;         // blocks
    const uint16_t *x;       // [rows][inner]
    uint16_t *xt;            // [inner][across]
    int inner, across;
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
        const int c = (int)(i - row * packs) * 8, live = min(8, a.cols - c);
        const long long from = row * a.cols + c;
        float g[8], u[8], dh[8];
        if constexpr (DT == PT_FLOAT32) {
            const S *kept = (const S *)a.kept + row * a.kept_pitch + c;
            gd_load<DT, 8>(kept, live, g);
            gd_load<DT, 8>(kept + a.kept_second, live, u);
        } else {
            gd_load_kept(a.kept, plane, 0, from, live, g);
            gd_load_kept(a.kept, plane, 1, from, live, u);
        }
        gd_load<GDT, 8>((const typename GE<GDT>::S *)a.grad + from, live, dh);
        S dg[8], du[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            float value, slope;
            gated_slope<DT != PT_FLOAT32>(a.act, g[k], value, slope);
            dg[k] = DType<DT>::from_c(k < live ? dh[k] * u[k] * slope : 0.0f);
            du[k] = DType<DT>::from_c(k < live ? dh[k] * value : 0.0f);
        }
        S *to = (S *)a.d + row * a.pitch + c;
        const int room = min(8, a.padded - c);
        if (room == 8) {
#pragma unroll
            for (int q = 0; q < 8 / GE<DT>::PK; q++) {
                *(gd_u32x4 *)(to + q * GE<DT>::PK) = *(gd_u32x4 *)(dg + q * GE<DT>::PK);
                *(gd_u32x4 *)(to + a.second + q * GE<DT>::PK) = *(gd_u32x4 *)(du + q * GE<DT>::PK);
            }
        } else {
            for (int k = 0; k < room; k++) {
                to[k] = dg[k];
                to[a.second + k] = du[k];
            }
        }
    }
}

// ------------------------------------------------------------- the calls
static int round8(int n) { return (n + 7) / 8 * 8; }
static unsigned grid_for(long long items) { return (unsigned)std::min<long long>((items + 255) / 256, 1 << 20); }

// Scratch of one call, given back in the stream's order.
struct GatedScratch {
    hipStream_t s;
    void *held[8];
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
    // fp32: two matrices side by side in down x 2 each elements
    pt_status beside(const float *a, const float *b, int rows, int cols, int down, int each, float **to)
    {
        PT_TRY(take((void **)to, (size_t)down * 2 * each * sizeof(float)));
        k_gated_beside<false><<<grid_for((long long)down * each), 256, 0, s>>>((float *)a, (float *)b, *to, rows, cols, down, each);
        return PT_OK;
    }
    // fp32 rows of `pitch`: themselves where they are, or a copy
    pt_status rows4(const float *a, long long rows, int cols, int pitch, const float **to)
    {
        *to = a;
        if (cols == pitch) return PT_OK;
        float *p = nullptr;
        PT_TRY(take((void **)&p, (size_t)rows * pitch * sizeof(float)));
        k_gated_pitch<<<grid_for(rows * pitch), 256, 0, s>>>(a, p, rows, cols, pitch);
        *to = p;
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

// fp32, more rows than k_gated_few takes: both weights lie side by side for
// one product, rather than two, where their rows fill no 16-byte packs (the
// product then reads whole packs of the copy, and runs the fp32 ring: 2048 x
// 1000 x 2731 214 us, 299 with two products in place), or where the tiles
// of one fill the CUs and twice as many take fewer rounds than two products
// do, which saves more than the copy costs (0.06 us a k against 3.2e-6 a
// weight: 2048 x 1024 x 2816 209 us, 256 with two).
struct GatedWide {
    int inner, outer;  // rounded up to whole packs
    bool beside;
    GatedWide(int M, int K, int F) : inner((K + 3) / 4 * 4), outer((F + 3) / 4 * 4)
    {
        const long long tiles = (long long)((M + 127) / 128) * ((F + 127) / 128);
        beside = inner != K || outer != F || (tiles >= 256 && 2 * ((tiles + 255) / 256) > (2 * tiles + 255) / 256 && F < 18750);
    }
    // the rows that both products are kept in, and where the second one's begin
    int pitch(int F) const { return beside ? 2 * outer : F; }
    long long second(int M, int F) const { return beside ? outer : (long long)M * F; }
};

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
    if (g.split > 1) launch_pair_join(g, DT, g.c1 ? GATED_KEPT : GATED_PRODUCT, s);
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
    if (d->dtype == PT_FLOAT32) {
        const GatedWide w(M, K, F);
        float *p = (float *)kept;
        if (!p) PT_TRY(scratch.take((void **)&p, (size_t)M * 2 * w.outer * sizeof(float)));
        if (w.beside) {
            float *weights = nullptr;
            const float *rows = nullptr;
            PT_TRY(scratch.beside((const float *)gate, (const float *)up, K, F, w.inner, w.outer, &weights));
            PT_TRY(scratch.rows4((const float *)x, M, K, w.inner, &rows));
            PT_TRY(product_f32(rows, w.inner, 1, weights, 2 * (size_t)w.outer, 1, p, M, 2 * w.outer, w.inner, stream));
        } else {
            PT_TRY(product_f32((const float *)x, K, 1, (const float *)gate, F, 1, p, M, F, K, stream));
            PT_TRY(product_f32((const float *)x, K, 1, (const float *)up, F, 1, p + n, M, F, K, stream));
        }
        k_gated_product<<<grid_for((long long)M * ((F + 3) / 4)), 256, 0, s>>>(p, (float *)h, M, F, w.pitch(F), w.second(M, F),
                                                                              d->activation);
        return PT_OK;
    }
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

static pt_status gated_backward_f32(const pt_gated_desc *d, const float *x, const float *gate, const float *up, const void *kept,
                                    const void *grad, float *dx, float *dgate, float *dup, GatedScratch &scratch, pt_stream_t stream)
{
    hipStream_t s = stream_of(stream);
    const int M = d->rows, K = d->inner, F = d->outer;
    const GatedWide w(M, K, F);
    const bool few = M <= kFewRows32 && F >= 4;  // (what k_gated_few kept lies in two planes)
    // dg and du side by side: one product takes both contractions of dx
    const size_t both_pitch = 2 * (size_t)w.outer;
    float *both = nullptr, *weights = nullptr;
    PT_TRY(scratch.take((void **)&both, M * both_pitch * sizeof(float)));
    SlopeArgs a = {kept, grad, both, w.outer, M, F, w.outer, 2 * w.outer, d->activation, few ? F : w.pitch(F),
                   few ? (long long)M * F : w.second(M, F), grid_for((long long)M * ((F + 7) / 8)), nullptr, nullptr, 0, 0};
    k_gated_slope<PT_FLOAT32, PT_FLOAT32><<<a.slopes, 256, 0, s>>>(a);
    if (dx && (long long)M * 4 < F && F % 4 == 0 && 16.0 * K * F > 1e8) {
        // few rows: two products and their sum move less than a copy of large
        // weights (33 x 4096 x 14336 both ways 546 us, 770 with the copy)
        float *other = nullptr;
        PT_TRY(scratch.take((void **)&other, (size_t)M * K * sizeof(float)));
        PT_TRY(product_f32(both, both_pitch, 1, gate, 1, F, dx, M, K, F, stream));
        PT_TRY(product_f32(both + w.outer, both_pitch, 1, up, 1, F, other, M, K, F, stream));
        k_gated_sum<<<grid_for((long long)M * K), 256, 0, s>>>(dx, other, (long long)M * K);
    } else if (dx) {
        PT_TRY(scratch.beside(gate, up, K, F, K, w.outer, &weights));
        PT_TRY(product_f32(both, both_pitch, 1, weights, 1, both_pitch, dx, M, K, 2 * w.outer, stream));
    }
    // both weights' gradients in one product where rows fill no packs, or
    // where one alone has fewer tiles than the GPU has CUs (4096 x 784 x
    // 1024: 149 us with the pass that takes them apart, 157 one after the other)
    if (dgate && (w.inner != K || w.outer != F || (long long)((K + 127) / 128) * ((F + 127) / 128) < 256)) {
        float *beside = nullptr;
        const float *rows = nullptr;
        PT_TRY(scratch.rows4(x, M, K, w.inner, &rows));
        PT_TRY(scratch.take((void **)&beside, w.inner * both_pitch * sizeof(float)));
        PT_TRY(product_f32(rows, 1, w.inner, both, both_pitch, 1, beside, w.inner, 2 * w.outer, M, stream));
        k_gated_beside<true><<<grid_for((long long)K * w.outer), 256, 0, s>>>(dgate, dup, beside, K, F, K, w.outer);
    } else if (dgate) {
        PT_TRY(product_f32(x, 1, K, both, both_pitch, 1, dgate, K, F, M, stream));
        PT_TRY(product_f32(x, 1, K, both + w.outer, both_pitch, 1, dup, K, F, M, stream));
    }
    return PT_OK;
}

static pt_status gated_backward_run(const pt_gated_desc *d, const void *x, const void *gate, const void *up, const void *kept,
                                    const void *grad, int grad_dtype, void *dx, void *dgate, void *dup, pt_stream_t stream)
{
    hipStream_t s = stream_of(stream);
    GatedScratch scratch(s);
    const int M = d->rows, K = d->inner, F = d->outer, pitch = round8(F);
    if (d->dtype == PT_FLOAT32)
        return gated_backward_f32(d, (const float *)x, (const float *)gate, (const float *)up, kept, grad, (float *)dx,
                                  (float *)dgate, (float *)dup, scratch, stream);
    uint16_t *dg = nullptr;
    const long long second = (long long)M * pitch;
    PT_TRY(scratch.take((void **)&dg, (size_t)second * 2 * 2));
    SlopeArgs a = {kept, grad, dg, second, M, F, pitch, pitch, d->activation, 0, 0, grid_for((long long)M * (pitch / 8)), nullptr, nullptr, 0, 0};
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
        pair_plan(g, false, tm);
        if (g.split > 1) PT_TRY(scratch.take((void **)&g.parts, (size_t)g.split * M * K * sizeof(float)));
        launch_pair_sum(g, d->dtype, tm, s);
    }
    if (dgate) {
        PairArgs g = {};
        g.a0 = a.xt;
        g.lda = g.K = a.across;
        g.kb = M;
        g.b0 = dg;
        g.b1 = dg + second;
        g.ldb = g.N = pitch;
        g.n_out = F;
        g.M = K;
        g.c1 = dgate;
        g.c2 = dup;
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
        if (d->dtype == PT_FLOAT32) PT_TRY(zeros(kept, PT_FLOAT32, 2 * (size_t)d->rows * ((d->outer + 3) / 4 * 4), stream));
        else PT_TRY(zeros(kept, PT_UINT8, 6 * n, stream));
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
