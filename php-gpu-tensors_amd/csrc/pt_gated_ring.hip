// Products over a pair of 16-bit matrices on gfx950's matrix cores, for the
// gated projection and its gradients (pt_gated.hip):
//   columns: P0 = A B0 and P1 = A B1, tiles of 256 x (128 + 128); a wave owns
//     the same 32 columns of both, so act(P0) P1 is taken from its registers.
//     The projection itself (A = x, B = gate, up), and both weights'
//     gradients (A = x transposed, B = dg, du) in one pass over A.
//   sum: P = A0 B0^T + A1 B1^T, one accumulator over both contractions: the
//     input's gradient (A = dg, du, B = gate, up as they lie).
// MFMA-bound: both run the ring of the plain whole-line product
// (pt_gemm_ring.hip): 8 waves in 2 x 4, A in 3 superstages of 64 k (whole
// 128-byte lines), B in 4 stages of 32 k, one barrier a step, a load to LDS
// between every few MFMAs, all reads' offsets immediate.  Tiles of 192 and 128
// rows (TM = 3, 2) serve where tiles of 256 leave CUs idle.  Edges cost
// nothing inside: rows and columns past
// the end read the last ones again and are not stored; past the
// contraction's end a lane's offset leaves the buffer's range, for which the
// buffer unit returns zeros, so what lies there (another row, or nothing) is
// neither read nor multiplied.  Few tiles: the contraction is split over
// workgroups, whose fp32 parts are added in order (k_pair_join).
// Measured, bfloat16, 8192 x 2048 x 8192 (550 GFLOP a call; the plain product
// at 8192^3 1170 TFLOP/s): both weights' gradients 432-450 us, the input's
// 432-442, the projection 530-555, of which 100 are its 537 MB of results and
// kept products: all workgroups of a round store at once, and nothing of the
// next round runs meanwhile, as the ring takes all of LDS.
#include "pt_gated.h"

#include <algorithm>

namespace pt {

constexpr int pair_bases(int stage_bytes, int max_inner)
{
    int s = 0;
    while (s * stage_bytes + max_inner < 65536) s++;
    return s;
}

constexpr uint32_t kPairRange = 0x7fffffffu, kPairOut = 0x80000000u;

// SUM: the sum form, else the columns form.
template <int DT, int TM, bool SUM, int STORE>
__global__ __launch_bounds__(512, 1) void k_pair(PairArgs g)
{
    using S = uint16_t;
    constexpr int NW = 8, WGN = 4, BK = 32, BM = 64 * TM, WTM = 32 * TM, TN = 2;
    constexpr int BN = SUM ? 256 : 128;    // output columns of a tile
    constexpr int NSA = 3, NSB = 4, PERIOD = 12, NS = 2;
    constexpr int SA_ELEMS = BM * 2 * BK;  // superstage: BM rows x 64 k
    constexpr int B_ELEMS = 256 * BK;
    // load instructions of a wave and step (192 rows: 12 of A, the last one
    // again by the waves that have none left, so that all wait for as many)
    constexpr int NQA = (BM + 127) / 128, NQB = 2, PER = NQA + NQB;
    constexpr int GROUP_M = 4;
    static_assert(TM >= 2 && TM <= 4, "load split");
    constexpr int SPA = pair_bases(SA_ELEMS * 2, (TM - 1) * 32 * 2 * BK * 2);
    constexpr int SPB = SUM ? pair_bases(B_ELEMS * 2, 32 * BK * 2) : pair_bases(B_ELEMS * 2, (16 + 4) * 128 * 2);
    static_assert(2 * SPA >= NSA && 2 * SPB >= NSB, "two bases cover the rings");
    __shared__ __attribute__((aligned(1024))) S lds_a[NSA * SA_ELEMS];
    __shared__ __attribute__((aligned(1024))) S lds_b[NSB * B_ELEMS];

    // neighbouring tiles on one XCD (workgroups go to the eight in turn)
    const int total = g.tiles_m * g.tiles_n, x = blockIdx.x % 8;
    const int t = x * (total / 8) + min(x, total % 8) + blockIdx.x / 8;
    const int group = t / (GROUP_M * g.tiles_n);
    const int first_m = group * GROUP_M;
    const int gsz = min(g.tiles_m - first_m, GROUP_M);
    const int in = t - group * GROUP_M * g.tiles_n;
    const int m0 = (first_m + in % gsz) * BM, n0 = in / gsz * BN;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WGN, wn = wave % WGN;

    // superstages of one matrix, and this split's share of all
    const int each = (g.K + 63) / 64, last = each - 1;
    const int s0 = blockIdx.y * g.stages, KS = min(g.stages, (SUM ? 2 : 1) * each - s0), KT = 2 * KS;
    const int tail = g.K - last * 64;  // k of the last superstage

    // A load (half h, instruction q4 of the wave): rows h * BM / 2 + 8 q ..,
    // lane L at row 8 q + L / 8, LDS position L % 8 holding chunk (L % 8) ^
    // swizzle.  In the last superstage the chunks past K are out of range.
    const S *A = (const S *)g.a0 + (long long)m0 * g.lda, *B = (const S *)g.b0 + (SUM ? (long long)n0 * g.ldb : 0);
    const long long to_a1 = SUM ? (const S *)g.a1 - (const S *)g.a0 : 0, to_b1 = (const S *)g.b1 - (const S *)g.b0;
    uint32_t offa[2][NQA], tail_a[2][NQA], offb[NQB], tail_b[2][NQB];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int q4 = 0; q4 < NQA; q4++) {
            const int row = h * (BM / 2) + min(wave * NQA + q4, BM / 16 - 1) * 8 + lane / 8, c = (lane % 8) ^ swz_k(row, 8);
            offa[h][q4] = (uint32_t)((long long)(min(m0 + row, g.M - 1) - m0) * g.lda + c * 8) * 2u;
            tail_a[h][q4] = c * 8 < tail ? offa[h][q4] : kPairOut;
        }
    if constexpr (SUM) {
        // B as A, in halves of a superstage: 256 rows x 64 bytes a step
#pragma unroll
        for (int q4 = 0; q4 < NQB; q4++) {
            const int row = (wave * NQB + q4) * 16 + lane / 4, c = (lane % 4) ^ swz_k(row, 4);
            offb[q4] = (uint32_t)((long long)(min(n0 + row, g.N - 1) - n0) * g.ldb + c * 8) * 2u;
            tail_b[0][q4] = c * 8 < tail ? offb[q4] : kPairOut;
            tail_b[1][q4] = 32 + c * 8 < tail ? offb[q4] : kPairOut;
        }
    } else {
        // B: each matrix 32 k-rows x 128 columns a step, a wave 4 rows of
        // both; 16-byte chunks XOR-swizzled by the row for the transposing reads
#pragma unroll
        for (int q4 = 0; q4 < NQB; q4++) {
            const int krow = wave * 4 + lane / 16, c = (lane % 16) ^ ((krow & 3) << 2);
            offb[q4] = (uint32_t)((long long)krow * g.ldb + min(n0 + c * 8, g.N - 8)) * 2u;
        }
    }
    // load IDX of issue step u, whose position in the period is J (u = J mod
    // 12; the prologue's u = -4 .. -1 are positions 8 .. 11).  Loads past the
    // share's end read its last stage again.
    auto issue_one = [&](int u, auto J, auto IDX) {
        constexpr int j = decltype(J)::value, idx = decltype(IDX)::value;
        if constexpr (idx < NQA) {
            constexpr int h = j & 1, slot = ((j + 4) >> 1) % NSA;
            const int s = s0 + min((u + 4) >> 1, KS - 1);
            const bool second = SUM && s >= each;
            const int sm = second ? s - each : s;
            buffer_load_lds16(A + ((second ? to_a1 : 0) + (long long)sm * 64), sm == last ? tail_a[h][idx] : offa[h][idx],
                              (PT_LDS_AS void *)(lds_a + slot * SA_ELEMS + (h * (BM / 2) + min(wave * NQA + idx, BM / 16 - 1) * 8) * 2 * BK),
                              kPairRange);
        } else {
            constexpr int q4 = idx - NQA, slot = (j + 3) % NSB;
            constexpr int half = (j + 3) & 1;  // of the superstage; kept where the last one is read again
            const int kb = 2 * s0 + min(u + 3, KT - 2 + half);
            if constexpr (SUM) {
                const bool second = kb >= 2 * each;
                const int km = second ? kb - 2 * each : kb;
                buffer_load_lds16(B + ((second ? to_b1 : 0) + (long long)km * BK), km >> 1 == last ? tail_b[half][q4] : offb[q4],
                                  (PT_LDS_AS void *)(lds_b + slot * B_ELEMS + (wave * NQB + q4) * 512), kPairRange);
            } else {
                // rows from kb on are out of the buffer's range
                const long long rest = max(0ll, (long long)(g.kb - kb * BK) * g.ldb * 2);
                buffer_load_lds16(B + ((q4 ? to_b1 : 0) + (long long)min(kb * BK, g.kb) * g.ldb), offb[q4],
                                  (PT_LDS_AS void *)(lds_b + slot * B_ELEMS + (q4 * NW + wave) * 512),
                                  (uint32_t)min(rest, (long long)kPairRange));
            }
        }
    };

    // fragment read bases, as in pt_gemm_ring.hip
    uint32_t abase[2][2][NS], bbase[2][2];  // B: [base][slice] (sum), [base][matrix] (columns)
    {
        const uint32_t la = (uint32_t)(size_t)(PT_LDS_AS const S *)lds_a;
        const uint32_t lb = (uint32_t)(size_t)(PT_LDS_AS const S *)lds_b;
        const int ra = wm * WTM + (lane & 31);
#pragma unroll
        for (int p = 0; p < 2; p++)
#pragma unroll
            for (int sl = 0; sl < NS; sl++) {
                const int kc = p * 4 + sl * 2 + (lane >> 5);
                abase[0][p][sl] = la + (uint32_t)(ra * 2 * BK + ((kc ^ swz_k(ra, 8)) << 3)) * 2u;
                abase[1][p][sl] = abase[0][p][sl] + (uint32_t)(SPA * SA_ELEMS * 2);
            }
        const int rb = wn * 64 + (lane & 31), grp = lane >> 4, s = lane & 15;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if constexpr (SUM) {
                const int kc = i * 2 + (lane >> 5);
                bbase[0][i] = lb + (uint32_t)(rb * BK + ((kc ^ swz_k(rb, 4)) << 3)) * 2u;
            } else {
                const int n = wn * 32 + (grp & 1) * 16 + 4 * (s & 3), kk = (grp >> 1) * 8 + (s >> 2);
                bbase[0][i] = lb + (uint32_t)(i * 128 * BK + kk * 128 + (((n >> 3) ^ ((kk & 3) << 2)) << 3) + (n & 7)) * 2u;
            }
            bbase[1][i] = bbase[0][i] + (uint32_t)(SPB * B_ELEMS * 2);
        }
    }

    floatx16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.0f;

    using Frag = typename FragT<DT>::type;
    // fragment q of slice SL of the step at period position J
    auto read_one = [&](auto J, auto SL, auto Q, Frag (&fa)[TM], Frag (&fb)[TN]) {
        constexpr int j = decltype(J)::value % PERIOD, sl = decltype(SL)::value, q = decltype(Q)::value;
        constexpr int slot = (j >> 1) % NSA, par = j & 1, ha = slot / SPA, sa = slot % SPA;
        constexpr int stb = j % NSB, hb = stb / SPB, sb = stb % SPB;
        if constexpr (q < TM) {
            lds_read_b128<(sa * SA_ELEMS + q * 32 * 2 * BK) * 2>(fa[q], abase[ha][par][sl]);
        } else if constexpr (SUM) {
            lds_read_b128<(sb * B_ELEMS + (q - TM) * 32 * BK) * 2>(fb[q - TM], bbase[hb][sl]);
        } else {
            s16x4_t h0, h1;
            lds_read_tr16<(sb * B_ELEMS + sl * 16 * 128) * 2>(h0, bbase[hb][q - TM]);
            lds_read_tr16<(sb * B_ELEMS + (sl * 16 + 4) * 128) * 2>(h1, bbase[hb][q - TM]);
            fb[q - TM] = __builtin_bit_cast(Frag, __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    };
    auto mfma_one = [&](auto Q, const Frag (&fa)[TM], const Frag (&fb)[TN]) {
        constexpr int q = decltype(Q)::value, i = q / TN, j = q % TN;
        if constexpr (DT == PT_BFLOAT16) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
        else acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[i], fb[j], acc[i][j], 0, 0, 0);
    };
    auto frag_wait = [&](Frag (&fa)[TM], Frag (&fb)[TN]) {
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (TM == 4)
            asm volatile("s_waitcnt lgkmcnt(0)"
                         : "+v"(fa[0]), "+v"(fa[1]), "+v"(fa[2]), "+v"(fa[3]), "+v"(fb[0]), "+v"(fb[1])::"memory");
        else if constexpr (TM == 3)
            asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(fa[0]), "+v"(fa[1]), "+v"(fa[2]), "+v"(fb[0]), "+v"(fb[1])::"memory");
        else asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(fa[0]), "+v"(fa[1]), "+v"(fb[0]), "+v"(fb[1])::"memory");
    };
    // the load issued at MFMA Q of slice SL of step kt: A's in slice 0, B's
    // in slice 1 (after the step's barrier)
    auto spread_load = [&](int kt, auto J, auto SL, auto Q) {
        constexpr int n = decltype(SL)::value == 0 ? NQA : NQB, every = TM * TN / n, q = decltype(Q)::value;
        if constexpr (q % every == 0) issue_one(kt, J, IC<(decltype(SL)::value == 0 ? 0 : NQA) + q / every>{});
    };

    // prologue: issue steps -4 .. -1 (A of superstages 0 and 1, B of steps
    // 0 .. 2); superstage 0 and B step 0 landed for everyone
    static_for<0, NQA>([&](auto Q) { issue_one(-4, IC<8>{}, Q); });
    static_for<0, PER>([&](auto Q) { issue_one(-3, IC<9>{}, Q); });
    static_for<0, PER>([&](auto Q) { issue_one(-2, IC<10>{}, Q); });
    static_for<0, PER>([&](auto Q) { issue_one(-1, IC<11>{}, Q); });
    ring_wait<2 * PER>();
    ring_barrier();
    Frag fa[2][TM], fb[2][TN];
    static_for<0, TM + TN>([&](auto Q) { read_one(IC<0>{}, IC<0>{}, Q, fa[0], fb[0]); });
    frag_wait(fa[0], fb[0]);
    for (int kt0 = 0; kt0 < KT; kt0 += PERIOD) {
        static_for<0, PERIOD>([&](auto J) {
            constexpr int j = decltype(J)::value;
            const int kt = kt0 + j;
            if (kt < KT) {  // uniform branch
                static_for<0, TM * TN>([&](auto Q) {
                    mfma_one(Q, fa[0], fb[0]);
                    if constexpr (decltype(Q)::value < TM + TN) read_one(J, IC<1>{}, Q, fa[1], fb[1]);
                    spread_load(kt, J, IC<0>{}, Q);
                    __builtin_amdgcn_sched_barrier(0);
                });
                frag_wait(fa[1], fb[1]);
                // in flight at most the loads of issue step kt - 1 and A's of
                // kt: those of kt - 2 (B of step kt + 1, superstage (kt + 1) / 2) landed
                ring_wait<PER + NQA>();
                ring_barrier();  // ... for everyone; step kt's stages are free
                static_for<0, TM * TN>([&](auto Q) {
                    mfma_one(Q, fa[1], fb[1]);
                    if constexpr (decltype(Q)::value < TM + TN) read_one(IC<j + 1>{}, IC<0>{}, Q, fa[0], fb[0]);
                    spread_load(kt, J, IC<1>{}, Q);
                    __builtin_amdgcn_sched_barrier(0);
                });
                frag_wait(fa[0], fb[0]);
            }
        });
    }
    ring_wait<0>();  // no load may still target LDS when the workgroup ends

    // In a 32 x 32 block lane l holds column l % 32 and rows 8 (e / 4) + 4 (l
    // / 32) + e % 4.  Each wave turns its blocks through its own part of LDS
    // (the ring is done with it), after which a lane holds 8 columns of a
    // row and stores 16 bytes.  A row of 40 floats keeps both halves of a
    // wave's writes, and a quarter's reads, on different banks.
    ring_barrier();
    constexpr int ROW = 40;
    static_assert(NW * 32 * ROW * 4 <= (int)sizeof(lds_a) && NW * 32 * ROW * 4 <= (int)sizeof(lds_b), "turned blocks fit");
    typedef float lds_float __attribute__((may_alias));
    typedef float lds_float4 __attribute__((ext_vector_type(4), may_alias));
    lds_float *box[2] = {(lds_float *)lds_a + wave * 32 * ROW, (lds_float *)lds_b + wave * 32 * ROW};
    auto turn = [&](const floatx16 &v, lds_float *to) {
#pragma unroll
        for (int e = 0; e < 16; e++) to[(8 * (e / 4) + 4 * (lane >> 5) + e % 4) * ROW + (lane & 31)] = v[e];
    };
    auto take = [&](const lds_float *from, int h, float (&v)[8]) {
        const lds_float4 *p = (const lds_float4 *)(from + (16 * h + lane / 4) * ROW + lane % 4 * 8);
        const lds_float4 a = p[0], b = p[1];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            v[k] = a[k];
            v[4 + k] = b[k];
        }
    };
    typedef uint32_t word4 __attribute__((ext_vector_type(4), aligned(2)));
    typedef uint32_t word2 __attribute__((ext_vector_type(2), aligned(1)));
    typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
    auto store16 = [&](void *c, long long at, int live, const float (&v)[8]) {
        word4 w;
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = pack_low<DT>(v[2 * k], v[2 * k + 1]);
        if (live >= 8) *(word4 *)((S *)c + at) = w;
        else
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k < live) ((S *)c)[at + k] = (S)(w[k / 2] >> (k & 1 ? 16 : 0));
    };
    auto store_kept = [&](int product, long long plane, long long at, int live, const float (&v)[8]) {
        S *high = (S *)((char *)g.c1 + kept_plane(plane, product, false)) + at;
        uint8_t *low = (uint8_t *)g.c1 + kept_plane(plane, product, true) + at;
        if (live >= 8) {
            word4 w;
            word2 l = {0, 0};
#pragma unroll
            for (int k = 0; k < 4; k++) w[k] = kept_high(v[2 * k]) | kept_high(v[2 * k + 1]) << 16;
#pragma unroll
            for (int k = 0; k < 8; k++) l[k / 4] |= kept_low(v[k]) << (8 * (k % 4));
            *(word4 *)high = w;
            *(word2 *)low = l;
        } else
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k < live) {
                    high[k] = (S)kept_high(v[k]);
                    low[k] = (uint8_t)kept_low(v[k]);
                }
    };
    const long long plane = (long long)g.M * g.n_out;
    float *parts = STORE == GATED_PARTS ? g.parts + (long long)blockIdx.y * (SUM ? 1 : 2) * plane : nullptr;
    // float16 gradients: multiplied back
    constexpr bool SHIFTED = DT == PT_FLOAT16 && (SUM ? STORE != GATED_PARTS : STORE == GATED_BOTH);
    int back[2][8];
    if constexpr (SHIFTED && !SUM)
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int n = min(n0 + wn * 32 + lane % 4 * 8 + k, g.n_out - 1);
            back[0][k] = -g.shift[n];
            back[1][k] = -g.shift[g.n_out + n];
        }
#pragma unroll
    for (int i = 0; i < TM; i++) {
        // (a wave's LDS accesses stay in order)
        turn(acc[i][0], box[0]);
        turn(acc[i][1], box[1]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int h = 0; h < 2; h++) {
            float p[8], q[8];
            take(box[0], h, p);
            take(box[1], h, q);
            const int m = m0 + wm * WTM + i * 32 + h * 16 + lane / 4;
            if (m >= g.M) continue;
            if constexpr (SHIFTED) {
                const int row = SUM ? -g.shift[m] : 0;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    p[k] = ldexpf(p[k], SUM ? row : back[0][k]);
                    q[k] = ldexpf(q[k], SUM ? row : back[1][k]);
                }
            }
#pragma unroll
            for (int j = 0; j < (SUM ? 2 : 1); j++) {
                const int n = n0 + (SUM ? wn * 64 + j * 32 : wn * 32) + lane % 4 * 8;
                const int live = g.n_out - n;
                if (live <= 0) continue;
                const long long at = (long long)m * g.n_out + n;
                if constexpr (STORE == GATED_PARTS) {
#pragma unroll
                    for (int part = 0; part < (SUM ? 1 : 2); part++) {
                        const float(&v)[8] = SUM ? (j ? q : p) : (part ? q : p);
                        float *to = parts + part * plane + at;
                        if (live >= 8) {
                            *(float4u *)to = float4u{v[0], v[1], v[2], v[3]};
                            *(float4u *)(to + 4) = float4u{v[4], v[5], v[6], v[7]};
                        } else
#pragma unroll
                            for (int k = 0; k < 8; k++)
                                if (k < live) to[k] = v[k];
                    }
                } else if constexpr (SUM) {
                    store16(g.c0, at, live, j ? q : p);
                } else if constexpr (STORE == GATED_BOTH) {
                    store16(g.c1, at, live, p);
                    store16(g.c2, at, live, q);
                } else {
                    if constexpr (STORE == GATED_KEPT) {
                        store_kept(0, plane, at, live, p);
                        store_kept(1, plane, at, live, q);
                    }
                    gated_products<true>(g.act, p, q);
                    store16(g.c0, at, live, p);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// Results from the parts of a split contraction, added in order; a thread
// takes 4 elements and has 4 parts of them on their way.
template <int DT, bool SUM, int STORE>
__global__ __launch_bounds__(256) void k_pair_join(PairArgs g)
{
    typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
    const long long plane = (long long)g.M * g.n_out, step = (SUM ? 1 : 2) * plane;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < plane; i += (long long)gridDim.x * 1024) {
        float4u p = {0.0f, 0.0f, 0.0f, 0.0f}, q = p;
        const int live = (int)min(4ll, plane - i);
        if (live == 4) {
#pragma unroll 4
            for (int k = 0; k < g.split; k++) {
                const float *from = g.parts + k * step + i;
                p += *(const float4u *)from;
                if (!SUM) q += *(const float4u *)(from + plane);
            }
        } else {
            for (int k = 0; k < g.split; k++)
                for (int e = 0; e < live; e++) {
                    const float *from = g.parts + k * step + i + e;
                    p[e] += from[0];
                    if (!SUM) q[e] += from[plane];
                }
        }
        if constexpr (DT == PT_FLOAT16 && (SUM || STORE == GATED_BOTH)) {
            long long row = i / g.n_out;
            int column = (int)(i - row * g.n_out);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (e >= live) continue;
                p[e] = ldexpf(p[e], -g.shift[SUM ? row : column]);
                if (!SUM) q[e] = ldexpf(q[e], -g.shift[g.n_out + column]);
                if (++column == g.n_out) column = 0, row++;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (e >= live) continue;
            if constexpr (SUM) {
                store_c<DT>(g.c0, (size_t)(i + e), p[e]);
            } else if constexpr (STORE == GATED_BOTH) {
                store_c<DT>(g.c1, (size_t)(i + e), p[e]);
                store_c<DT>(g.c2, (size_t)(i + e), q[e]);
            } else {
                if constexpr (STORE == GATED_KEPT) gated_keep<DT>(g.c1, plane, i + e, p[e], q[e]);
                store_c<DT>(g.c0, (size_t)(i + e), gated_act<DT != PT_FLOAT32>(g.act, p[e]) * q[e]);
            }
        }
    }
}

// The tile's rows and the split of the contraction that are estimated to take
// the least time, from what was measured on this GPU: a step of 32 k takes a
// workgroup of 256, 192 and 128 rows 0.65, 0.58 and 0.5 us where few run, as
// long as its loads take from HBM, and 0.9, 0.7 and 0.5 us where all CUs run
// (0.6 at least where one row of tiles shares none of B); HBM gives 5 TB/s; a
// split writes and reads fp32 parts and joins them in a second kernel, 4 us.
void pair_plan(PairArgs &g, bool columns, int &tm)
{
    const int bn = columns ? 128 : 256, all = (columns ? 1 : 2) * ((g.K + 63) / 64);
    const long long across = (g.n_out + bn - 1) / bn;
    const double plane = (columns ? 2.0 : 1.0) * g.M * g.n_out;
    const double hbm = (2.0 * g.K * g.n_out + (columns ? 1.0 : 2.0) * g.M * g.K) * 2 / 5e6;  // us
    double best = 0;
    g.split = 0;
    for (int t = 4; t >= 2; t--)
        for (int parts = 1; parts <= 32; parts *= 2) {
            const int stages = (all + parts - 1) / parts, split = (all + stages - 1) / stages;
            if (split > 1 && stages < 2) break;
            const long long down = (g.M + 64 * t - 1) / (64 * t), groups = down * across * split;
            const double full = std::min(1.0, (double)groups / 256);
            const double step = t == 4 ? 0.65 + 0.25 * full : t == 3 ? 0.58 + 0.12 * full : down == 1 ? 0.6 : 0.5;
            double time = std::max((double)((groups + 255) / 256) * 2 * stages * step, hbm);
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

template <int DT, bool SUM, int STORE>
static void join_parts(const PairArgs &g, hipStream_t s)
{
    const unsigned blocks = (unsigned)std::min<long long>(((long long)g.M * g.n_out + 1023) / 1024, 1 << 20);
    k_pair_join<DT, SUM, STORE><<<blocks, 256, 0, s>>>(g);
}

void launch_pair_join(const PairArgs &g, int dtype, bool sum, int store, hipStream_t s)
{
    auto go = [&](auto DTC) {
        constexpr int D = decltype(DTC)::value;
        if (store == GATED_PRODUCT) join_parts<D, false, GATED_PRODUCT>(g, s);
        else join_parts<D, false, GATED_KEPT>(g, s);
    };
    if (dtype == PT_BFLOAT16) go(IC<PT_BFLOAT16>{});
    else if (dtype == PT_FLOAT16) go(IC<PT_FLOAT16>{});
    else if (sum) join_parts<PT_FLOAT32, true, GATED_PRODUCT>(g, s);
    else if (store == GATED_BOTH) join_parts<PT_FLOAT32, false, GATED_BOTH>(g, s);
    else go(IC<PT_FLOAT32>{});
}

template <int DT, bool SUM, int STORE>
static void launch_pair_store(const PairArgs &g, int tm, hipStream_t s)
{
    const dim3 grid(g.tiles_m * g.tiles_n, g.split);
    if (g.split > 1) {
        if (tm == 4) k_pair<DT, 4, SUM, GATED_PARTS><<<grid, 512, 0, s>>>(g);
        else if (tm == 3) k_pair<DT, 3, SUM, GATED_PARTS><<<grid, 512, 0, s>>>(g);
        else k_pair<DT, 2, SUM, GATED_PARTS><<<grid, 512, 0, s>>>(g);
        join_parts<DT, SUM, STORE>(g, s);
        return;
    }
    if (tm == 4) k_pair<DT, 4, SUM, STORE><<<grid, 512, 0, s>>>(g);
    else if (tm == 3) k_pair<DT, 3, SUM, STORE><<<grid, 512, 0, s>>>(g);
    else k_pair<DT, 2, SUM, STORE><<<grid, 512, 0, s>>>(g);
}

void launch_pair_columns(const PairArgs &g, int dtype, int tm, int store, hipStream_t s)
{
    auto go = [&](auto DTC) {
        constexpr int D = decltype(DTC)::value;
        if (store == GATED_PRODUCT) launch_pair_store<D, false, GATED_PRODUCT>(g, tm, s);
        else if (store == GATED_KEPT) launch_pair_store<D, false, GATED_KEPT>(g, tm, s);
        else launch_pair_store<D, false, GATED_BOTH>(g, tm, s);
    };
    if (dtype == PT_BFLOAT16) go(IC<PT_BFLOAT16>{});
    else go(IC<PT_FLOAT16>{});
}

void launch_pair_sum(const PairArgs &g, int dtype, int tm, hipStream_t s)
{
    if (dtype == PT_BFLOAT16) launch_pair_store<PT_BFLOAT16, true, GATED_PRODUCT>(g, tm, s);
    else launch_pair_store<PT_FLOAT16, true, GATED_PRODUCT>(g, tm, s);
}

}  // namespace pt
