// Products over a pair of fp32 matrices on gfx950's matrix cores, for the
// gated projection and its gradients of more rows than k_gated_few takes
// (pt_gated.hip):
//   columns: P0 = A B0 and P1 = A B1, a wave owns the same 32 columns of
//     both, so act(P0) P1 is taken from its registers; A as it lies (the
//     projection itself), or transposed (both weights' gradients in one pass
//     over x).
//   sum: P = A0 B0^T + A1 B1^T, one accumulator over both contractions (the
//     input's gradient).
// MFMA-bound: 256 flops a cycle and CU.  A workgroup's 4 waves own a tile of
// 32 TM x 128 in 16 x 16 blocks, A and B each 16 k deep in LDS twice: while
// one stage is multiplied (64 MFMAs of 32 cycles at TM = 4), the next comes
// from memory through registers.  Two workgroups a CU and more fill each
// other's waits.  All operands are read in place, in packs of 4 elements at
// any address; a contraction's last pack, where it is not whole, by elements.
// Rows past the end read the last one again, columns past it the next row's,
// and neither is stored; past the contraction's end both operands are zeros.
// Measured: 4096 x 784 x 1024, the projection with its products kept, 126 us (104
// TFLOP/s; two plain products and a pass over both 133); both ways 155 x
// 2080 x 160 43 us and 300 x 501 x 601 57 (84 and 82 with plain products and the copies
// that they want).  The matrix cores are busy for 80 % of a long
// contraction: LDS reads and writes beside fp32 MFMAs take their time, be
// the blocks of 16 or 32, the barrier in the middle of a stage, or one to four
// workgroups on a CU.
#include "pt_gated.h"

#include <algorithm>

namespace pt {

constexpr int kWideK = 16, kWideColumns = 128, kWideThreads = 256;

// A tile of ROWS rows (or columns) by 16 k of an operand.  ALONG: k is
// contiguous in memory; a row's 4 packs lie in LDS in an order turned by the
// row, so that the reads of 16 rows' packs spread over the banks.  Else rows
// of k, 4 elements longer than needed, so that the k that a wave reads
// together, 4 apart, lie on different banks.
template <int ROWS, bool ALONG>
struct WideTile {
    static constexpr bool IS_ALONG = ALONG;
    static constexpr int PITCH = ALONG ? kWideK : ROWS + 4, FLOATS = ALONG ? ROWS * kWideK : kWideK * PITCH;
    static constexpr int ITEMS = ROWS * 4, EACH = (ITEMS + kWideThreads - 1) / kWideThreads;
    __device__ static int row(int item) { return ALONG ? item / 4 : item / (ROWS / 4); }      // (ALONG: row, else k)
    __device__ static int pack(int item) { return (ALONG ? item % 4 : item % (ROWS / 4)) * 4; }  // (ALONG: k, else column)
    __device__ static int place(int item)
    {
        const int r = row(item), p = pack(item);
        return ALONG ? r * PITCH + (p ^ ((r >> 1 & 3) << 2)) : r * PITCH + p;
    }
    // the 4 k from 4 quarter on of a row
    __device__ static floatx4 take(const float *tile, int r, int quarter)
    {
        if constexpr (ALONG) return *(const floatx4 *)(tile + r * PITCH + ((quarter ^ (r >> 1 & 3)) << 2));
        else {
            const float *p = tile + quarter * 4 * PITCH + r;
            return floatx4{p[0], p[PITCH], p[2 * PITCH], p[3 * PITCH]};
        }
    }
};

// Loads at a lane's byte offset (a multiple of 4) from a wave-uniform base;
// the buffer unit returns zeros for each element from `range` on.
constexpr uint32_t kWideRange = 0x7fffffffu, kWideOut = 0x80000000u;
__device__ __forceinline__ floatx4 wide_pack(const float *base, uint32_t range, uint32_t off)
{
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(base), (short)0, (int)range, 0x00020000);
    return __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}
// element by element, zeros from the `live`-th on
__device__ __forceinline__ floatx4 wide_each(const float *base, uint32_t off, int live)
{
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(base), (short)0, (int)kWideRange, 0x00020000);
    floatx4 v;
#pragma unroll
    for (int i = 0; i < 4; i++)
        v[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, (int)(i < live ? off + 4 * i : kWideOut), 0, 0));
    return v;
}

template <int TM, int FORM>
__global__ __launch_bounds__(kWideThreads, 2) void k_wide(PairArgs g)
{
    constexpr bool SUM = FORM == WIDE_SUM, A_ALONG = FORM != WIDE_TURNED;
    constexpr int BM = 32 * TM, BN = SUM ? kWideColumns : kWideColumns / 2, GROUP_M = 4;
    using TA = WideTile<BM, A_ALONG>;
    using TB = WideTile<BN, SUM>;
    constexpr int NB = SUM ? 1 : 2;  // B's tiles, of each matrix
    __shared__ __attribute__((aligned(16))) float lds_a[2][TA::FLOATS], lds_b[2][NB][TB::FLOATS];

    // neighbouring tiles on one XCD (workgroups go to the eight in turn)
    const int total = g.tiles_m * g.tiles_n, x = blockIdx.x % 8;
    const int t = x * (total / 8) + min(x, total % 8) + blockIdx.x / 8;
    const int group = t / (GROUP_M * g.tiles_n), first_m = group * GROUP_M;
    const int gsz = min(g.tiles_m - first_m, GROUP_M), in = t - group * GROUP_M * g.tiles_n;
    const int m0 = (first_m + in % gsz) * BM, n0 = in / gsz * BN;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;

    // stages of one matrix, and this split's share of all
    const int each = (g.K + kWideK - 1) / kWideK;
    const int s0 = blockIdx.y * g.stages, KS = min(g.stages, (SUM ? 2 : 1) * each - s0);

    // An operand's tile, of rows (columns) from r0 on of `rows`, and its lanes'
    // byte offsets from the tile's first element of a stage.
    auto offsets = [&](auto T, int r0, int rows, long long ld, uint32_t (&off)[decltype(T)::EACH]) {
        using Tile = decltype(T);
#pragma unroll
        for (int e = 0; e < Tile::EACH; e++) {
            const int r = Tile::row(tid + e * kWideThreads), p = Tile::pack(tid + e * kWideThreads);
            off[e] = (uint32_t)((long long)(Tile::IS_ALONG ? min(r0 + r, rows - 1) - r0 : r) * ld + p) * 4u;
        }
    };
    uint32_t offa[TA::EACH], offb[TB::EACH];
    offsets(TA{}, m0, g.M, g.lda, offa);
    offsets(TB{}, n0, g.N, g.ldb, offb);
    auto fetch = [&](auto T, const float *p, int r0, int rows, long long ld, int k0, const uint32_t (&off)[decltype(T)::EACH],
                     floatx4 (&to)[decltype(T)::EACH]) {
        using Tile = decltype(T);
        constexpr bool ALONG = Tile::IS_ALONG;
        // past the contraction's end, along: the offset leaves the range; else the rows do
        const float *base = p + (ALONG ? r0 * ld + k0 : k0 * ld + r0);
        const uint32_t range = (uint32_t)min(((g.K - k0) * ld - r0) * 4, (long long)kWideRange);
        // (no vector instruction but the loads themselves where the stage is whole:
        // beside fp32 MFMAs each one takes their time)
        const bool whole = !ALONG || k0 + kWideK <= g.K;
#pragma unroll
        for (int e = 0; e < Tile::EACH; e++) {
            const int item = tid + e * kWideThreads;
            if (Tile::ITEMS % kWideThreads && item >= Tile::ITEMS) continue;
            if (whole) to[e] = wide_pack(base, ALONG ? kWideRange : range, off[e]);
            else to[e] = wide_each(base, off[e], g.K - k0 - Tile::pack(item));  // a pack may reach past the row
        }
    };
    floatx4 ra[TA::EACH], rb[NB][TB::EACH];
    auto load = [&](int s) {
        const bool second = SUM && s >= each;
        const int k0 = (second ? s - each : s) * kWideK;
        fetch(TA{}, (const float *)(second ? g.a1 : g.a0), m0, g.M, g.lda, k0, offa, ra);
        fetch(TB{}, (const float *)(second ? g.b1 : g.b0), n0, g.N, g.ldb, k0, offb, rb[0]);
        if constexpr (!SUM) fetch(TB{}, (const float *)g.b1, n0, g.N, g.ldb, k0, offb, rb[1]);
    };
    auto put = [&](int half) {
#pragma unroll
        for (int e = 0; e < TA::EACH; e++) {
            const int item = tid + e * kWideThreads;
            if (TA::ITEMS % kWideThreads && item >= TA::ITEMS) continue;
            *(floatx4 *)(lds_a[half] + TA::place(item)) = ra[e];
        }
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < TB::EACH; e++) *(floatx4 *)(lds_b[half][b] + TB::place(tid + e * kWideThreads)) = rb[b][e];
    };

    const int col = lane & 15, quarter = lane >> 4;
    // a wave's 4 blocks of 16 columns: 64 of the tile's (sum), or 32 of each matrix
    auto block = [&](int j) { return SUM ? wn * 64 + j * 16 : wn * 32 + (j & 1) * 16; };
    floatx4 acc[TM][4];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

    load(s0);
    put(0);
    __syncthreads();
    auto stage = [&](int s, auto HALF) {
        constexpr int h = decltype(HALF)::value;
        if (s + 1 < KS) load(s0 + s + 1);
        floatx4 fa[TM], fb[4];
#pragma unroll
        for (int i = 0; i < TM; i++) fa[i] = TA::take(lds_a[h], wm * 16 * TM + i * 16 + col, quarter);
#pragma unroll
        for (int j = 0; j < 4; j++) fb[j] = TB::take(lds_b[h][SUM ? 0 : j >> 1], block(j) + col, quarter);
        __builtin_amdgcn_sched_barrier(0);
        // (the transposed block: a lane then holds 4 columns of a row)
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[j][k], fa[i][k], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (s + 1 < KS) put(1 - h);  // (nobody reads that half since the last barrier)
        __syncthreads();
    };
    for (int s = 0; s < KS; s += 2) {
        stage(s, IC<0>{});
        if (s + 1 < KS) stage(s + 1, IC<1>{});
    }

    typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
    auto store = [&](float *to, int live, const floatx4 &v) {
        if (live >= 4) *(float4u *)to = v;
        else
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (e < live) to[e] = v[e];
    };
    const long long plane = (long long)g.M * g.n_out;
    float *parts = g.split > 1 ? g.parts + (long long)blockIdx.y * (SUM ? 1 : 2) * plane : nullptr;
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int m = m0 + wm * 16 * TM + i * 16 + col;
        if (m >= g.M) continue;
#pragma unroll
        for (int j = 0; j < (SUM ? 4 : 2); j++) {
            const int n = n0 + block(j) + quarter * 4, live = g.n_out - n;
            if (live <= 0) continue;
            const long long at = (long long)m * g.n_out + n;
            const floatx4 &p = acc[i][j], &q = acc[i][j ^ 2];
            if constexpr (SUM) {
                store((parts ? parts : (float *)g.c0) + at, live, p);
            } else {
                // both products: the gradients, what the gradient keeps, or parts
                float *first = parts ? parts : (float *)g.c1, *other = parts ? parts + plane : FORM == WIDE_TURNED ? (float *)g.c2 : first + plane;
                if (first) {
                    store(first + at, live, p);
                    store(other + at, live, q);
                }
                if (FORM == WIDE_TURNED || parts) continue;
                float v[4] = {p[0], p[1], p[2], p[3]};
                const float u[4] = {q[0], q[1], q[2], q[3]};
                gated_products<false>(g.act, v, u);
                store((float *)g.c0 + at, live, floatx4{v[0], v[1], v[2], v[3]});
            }
        }
    }
}

// The tile's rows and the split of the contraction that are estimated to take
// the least time: a workgroup's stage of 16 k takes 0.24 us for each 32 rows,
// its beginning and end 2 us, a CU's workgroups share it, and one that is alone
// on its CU waits 0.2 us more a stage; a split writes and reads fp32 parts
// and joins them in a second kernel, 4 us.  (A closer model of what a CU's
// workgroups hide from each other chose worse for small sizes: 155 x 2080 x 160
// both ways 43 us with this one, 54 with that.)
void wide_plan(PairArgs &g, int form, int &tm)
{
    const bool columns = form != WIDE_SUM;
    const int bn = columns ? kWideColumns / 2 : kWideColumns, all = (columns ? 1 : 2) * ((g.K + kWideK - 1) / kWideK);
    const long long across = (g.n_out + bn - 1) / bn;
    const double plane = (columns ? 2.0 : 1.0) * g.M * g.n_out;
    double best = 0;
    g.split = 0;
    for (int t = 5; t >= 2; t--)
        for (int parts = 1; parts <= 64; parts++) {
            const int stages = (all + parts - 1) / parts, split = (all + stages - 1) / stages;
            if (split != parts) continue;
            if (split > 1 && stages < 4) break;
            const long long down = (g.M + 32 * t - 1) / (32 * t), each = (down * across * split + 255) / 256;  // of a CU
            double time = (double)each * (stages * 0.24 * t + 2.0) + (each == 1 ? stages * 0.2 : 2.0);
            if (split > 1) time += 4.0 + split * plane * 8 / 5e6;
            if (g.split && time >= best) continue;
            best = time;
            tm = t;
            g.split = split;
            g.stages = stages;
            g.tiles_m = (int)down;
        }
    g.tiles_n = (int)across;
}

template <int FORM>
static void launch_form(const PairArgs &g, int tm, hipStream_t s)
{
    const dim3 grid(g.tiles_m * g.tiles_n, g.split);
    if (tm == 5) k_wide<5, FORM><<<grid, kWideThreads, 0, s>>>(g);
    else if (tm == 4) k_wide<4, FORM><<<grid, kWideThreads, 0, s>>>(g);
    else if (tm == 3) k_wide<3, FORM><<<grid, kWideThreads, 0, s>>>(g);
    else k_wide<2, FORM><<<grid, kWideThreads, 0, s>>>(g);
}

void launch_wide(const PairArgs &g, int tm, int form, int store, hipStream_t s)
{
    if (form == WIDE_COLUMNS) launch_form<WIDE_COLUMNS>(g, tm, s);
    else if (form == WIDE_TURNED) launch_form<WIDE_TURNED>(g, tm, s);
    else launch_form<WIDE_SUM>(g, tm, s);
    if (g.split > 1) launch_pair_join(g, PT_FLOAT32, form == WIDE_SUM, store, s);
}

}  // namespace pt
