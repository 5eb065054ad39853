// Log probabilities of given tokens, with the entropy and the likeliest
// alternatives of each row, and their gradients, for gfx950.  Of a row x
// with maximum m:
//   s = sum e^(x - m),  log p_j = x_j - m - log s
//   H = -sum p_j log p_j = log s + (1 / s) sum (m - x_j) e^(x_j - m)
// The row is read once: each thread keeps a running m, s and the second sum
// t over its elements and rescales them where its maximum rises
// (t' = (t + d s) e^-d and s' = s e^-d for m' = m + d); every term of H is
// positive, so nothing cancels.  m and log s are kept apart for the gradient:
// their sum would lose log s in a row masked by the type's lowest value.
// HBM-bound; an element takes about 9 vector instructions and one exponential:
// 4096 rows of 32768 float32 scores 82 us (6.5 TB/s), 2000 rows of 50021 in
// bfloat16 36 us (5.6 TB/s).
//
// The likeliest `top` elements come from the same read.  A wave holds the
// best it has seen in order, one a lane; a pack of elements is compared with
// the worst of them by its maximum, which the running maximum needs anyway,
// so on a row without order almost no pack is looked at again (about k (1 +
// ln(n / k)) insertions of n elements).  The waves tell each other how large
// their best are, so that each lists its share only.  Equal values: the lower
// index first.  With 8 alternatives the bfloat16 rows above take 59 us, bound
// by the search's instructions; the float32 rows of that width 73 against 67.
//
// Gradient, for upstream a of log p_token, h of H and u_i of the log
// probability of alternative i:
//   dx_j = [j = token] a + sum_i [j = i] u_i
//          - p_j (a + sum u_i) - h p_j (log p_j + H)
// One read and one write: 200 us for the float32 scores above (5.4 TB/s).
#include "pt_common.h"

#include <algorithm>
#include <limits.h>

namespace pt {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

typedef unsigned int lp_u32x4 __attribute__((ext_vector_type(4), aligned(1)));

template <int DT> struct LpPack {
    using S = typename DType<DT>::S;
    static constexpr int V = 16 / sizeof(S);
    // 16 bytes at any element boundary; read once
    __device__ __forceinline__ static lp_u32x4 load(const S *p)
    {
        return __builtin_nontemporal_load((const lp_u32x4 *)p);
    }
    __device__ __forceinline__ static void widen(const lp_u32x4 &raw, float (&v)[V])
    {
        union { lp_u32x4 raw; S s[V]; } u;
        u.raw = raw;
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = DType<DT>::to_c(u.s[i]);
    }
    // elements that add nothing
    __device__ __forceinline__ static lp_u32x4 nothing()
    {
        const uint32_t low = sizeof(S) == 4 ? 0xff800000u : DT == PT_FLOAT16 ? 0xfc00fc00u : 0xff80ff80u;
        return lp_u32x4{low, low, low, low};
    }
    // element `at`, if it is one of these, becomes a NaN
    __device__ __forceinline__ static void drop(lp_u32x4 &raw, int at)
    {
        if constexpr (sizeof(S) == 4) {
#pragma unroll
            for (int i = 0; i < 4; i++) raw[i] = at == i ? 0x7fffffffu : raw[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) raw[i] |= (at >> 1) == i ? (at & 1 ? 0x7fff0000u : 0x7fffu) : 0u;
        }
    }
};

// Running maximum, sum and entropy sum.
struct LpSum {
    float m, s, t;
    __device__ __forceinline__ void init() { m = -INFINITY, s = 0.0f, t = 0.0f; }
    __device__ __forceinline__ void rise(float to)
    {
        if (to > m) {
            // past e^-150 the factor is 0, and a longer way would only overflow beside it
            const float d = fminf(to - m, 150.0f), f = __builtin_amdgcn_exp2f(-d * kLog2e);
            t = (t + d * s) * f;
            s *= f;
            m = to;
        }
    }
    __device__ __forceinline__ float ref() const { return m == -INFINITY ? 0.0f : m; }
    // x <= m, or NaN; past e^-150 the exponential is 0 and the logarithm
    // beside it is cut, so that -inf adds nothing (a NaN stays in s)
    __device__ __forceinline__ void add(float x, float r)
    {
        const float y = x - r, e = __builtin_amdgcn_exp2f(y * kLog2e);
        s += e;
        t = fmaf(-fmaxf(y, -150.0f), e, t);
    }
    __device__ __forceinline__ void join(const LpSum &o)
    {
        const float to = fmaxf(m, o.m);
        if (to == -INFINITY) {
            s += o.s;  // no maximum: both 0, or NaN
            t += o.t;
            return;
        }
        LpSum b = o;
        rise(to);
        b.rise(to);
        s += b.s;
        t += b.t;
    }
};

// The top-th largest of the lanes' values: of elements of which these are
// some, the top-th largest is no smaller.  NaN counts as -inf.
__device__ __forceinline__ float lp_bound(float x, int top)
{
    float y = x > -INFINITY ? x : -INFINITY, m;
    for (int have = 0;;) {
        m = wave_all(y, FMax{});
        have += (int)__popcll(__ballot(y == m));
        if (have >= top) return m;  // at the latest where all are -inf
        y = y == m ? -INFINITY : y;
    }
}

// The best `top` elements of a wave, in lanes 0 .. top - 1.
struct LpTop {
    float v, worst, floor;  // worst: what an element has to reach, at least floor
    int i, worst_i;
    // no element below `x` is wanted
    __device__ __forceinline__ void at_least(float x)
    {
        floor = fmaxf(floor, x);
        if (floor > worst) {
            worst = floor;
            worst_i = INT_MAX;
        }
    }
    __device__ __forceinline__ void init()
    {
        v = worst = floor = -INFINITY;
        i = worst_i = INT_MAX;
    }
    __device__ __forceinline__ static bool better(float a, int ai, float b, int bi) { return a > b || (a == b && ai < bi); }
    // every lane offers one element (index INT_MAX: none)
    __device__ __forceinline__ void offer(float x, int at, int top, int lane)
    {
        bool want = better(x, at, worst, worst_i);
        for (uint64_t left = __ballot(want); left; left = __ballot(want)) {
            const int from = (int)__builtin_ctzll(left);
            const float cx = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), from));
            const int ci = __builtin_amdgcn_readlane(at, from);
            const int place = (int)__popcll(__ballot(lane < top && better(v, i, cx, ci)));
            // the lane before: one DPP move each (wave_shr:1)
            const float up = __builtin_bit_cast(
                float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x138, 0xF, 0xF, false));
            const int up_i = __builtin_amdgcn_update_dpp(0, i, 0x138, 0xF, 0xF, false);
            if (lane >= place) {
                v = lane == place ? cx : up;
                i = lane == place ? ci : up_i;
            }
            const int last_i = __builtin_amdgcn_readlane(i, top - 1);
            const float last = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), top - 1));
            if (last_i != INT_MAX && last >= floor) {  // the list is full: its last bounds what follows
                worst = last;
                worst_i = last_i;
            }
            want = lane != from && want && better(x, at, worst, worst_i);
        }
    }
};

struct LpArgs {
    const void *x;
    long long stride;
    int rows, classes, splits, top;
    const int32_t *tokens;
    float *logprob, *entropy, *stats, *top_v;
    int32_t *top_i;
    float *part;  // [row][split][3 + 2 top]
};

__device__ __forceinline__ LpSum lp_wave(LpSum a)
{
    const float m = wave_all(a.m, FMax{});
    if (m != -INFINITY) a.rise(m);
    a.m = m;
    a.s = wave_all(a.s, FAdd{});
    a.t = wave_all(a.t, FAdd{});
    return a;
}

// The score of the row's token, asked for before the row is read: 0 where
// there is none, NaN past the classes.
template <int DT>
__device__ __forceinline__ float lp_token(const LpArgs &g, int row, bool &named)
{
    named = false;
    if (!g.logprob) return 0.0f;
    const int tok = g.tokens[row];
    if (tok < 0) return 0.0f;
    named = true;
    if (tok >= g.classes) return __builtin_nanf("");
    return DType<DT>::to_c(((const typename DType<DT>::S *)g.x)[(long long)row * g.stride + tok]);
}

// One wave writes a row's results.
__device__ __forceinline__ void lp_finish(const LpArgs &g, int row, const LpSum &a, const LpTop &top, float token, bool named,
                                          int lane)
{
    // a row of -inf alone: no element has a probability
    const bool none = a.m == -INFINITY && a.s == 0.0f;
    const float r = a.ref(), log_s = __builtin_amdgcn_logf(a.s) * kLn2;
    if (lane == 0) {
        if (g.stats) {
            g.stats[2 * (long long)row] = a.m;
            g.stats[2 * (long long)row + 1] = log_s;
        }
        if (g.entropy) g.entropy[row] = none ? 0.0f : log_s + a.t / a.s;
        // (a NaN token score stays one in a row without probabilities)
        if (g.logprob) g.logprob[row] = !named ? 0.0f : none && token == token ? -INFINITY : token - r - log_s;
    }
    if (lane < g.top) {
        const long long at = (long long)row * g.top + lane;
        if (g.top_v) g.top_v[at] = none ? -INFINITY : top.v - r - log_s;
        if (g.top_i) g.top_i[at] = top.i == INT_MAX ? -1 : top.i;  // fewer than `top` elements that are no NaN
    }
}

// A row, or the part blockIdx.y of it, by NW waves.
template <int DT, int NW, bool TOP>
__global__ __launch_bounds__(64 * NW, 8) void k_logprobs(LpArgs g)
{
    using P = LpPack<DT>;
    // Packs in flight a lane.  Four of 16 bits and the search need more than
    // the 64 registers of eight waves a SIMD: 69 us with what spills, 60 with
    // three (2000 rows of 50021, top 8).
    constexpr int V = P::V, UN = TOP && V == 8 ? 3 : 4;
    __shared__ float box[NW][3];
    __shared__ float top_v[TOP ? NW : 1][64];
    __shared__ int top_i[TOP ? NW : 1][64];
    __shared__ float best_v[64];
    __shared__ int best_i[64];
    __shared__ volatile float share[TOP ? NW : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.x;
    const typename P::S *x = (const typename P::S *)g.x + (long long)row * g.stride;
    const int per = g.splits > 1 ? ((g.classes + g.splits - 1) / g.splits + V * 64 - 1) / (V * 64) * (V * 64) : g.classes;
    const int begin = min((long long)g.classes, (long long)per * blockIdx.y), end = min((long long)g.classes, (long long)begin + per);

    bool named = false;
    const float token = g.splits == 1 ? lp_token<DT>(g, row, named) : 0.0f;
    LpSum a;
    a.init();
    LpTop top;
    top.init();
    // What the waves tell each other: a value that `deep` of a wave's elements
    // reach; where `wide` waves reach a value, `top` elements do.
    const int deep = TOP ? (g.top + NW - 1) / NW : 0, wide = TOP ? (g.top + deep - 1) / deep : 0;
    int calls = 0;
    const int turn = NW * 64 * V;
    // NP packs at once; `in`: this lane's are inside (all lanes' if NP > 1)
    auto take = [&](int at, bool in, auto NP) __attribute__((always_inline)) {
        constexpr int np = decltype(NP)::value;
        lp_u32x4 raw[np];
        float v[np][V];
#pragma unroll
        for (int p = 0; p < np; p++) {
            if (np > 1 || in) raw[p] = P::load(x + at + p * turn);
            else raw[p] = P::nothing();
        }
#pragma unroll
        for (int p = 0; p < np; p++) P::widen(raw[p], v[p]);
        float each[np], most = __builtin_nanf("");
#pragma unroll
        for (int p = 0; p < np; p++) {
            each[p] = v[p][0];
#pragma unroll
            for (int k = 1; k < V; k++) each[p] = fmaxf(each[p], v[p][k]);
            most = fmaxf(most, each[p]);
        }
        a.rise(most);
        const float r = a.ref();
#pragma unroll
        for (int p = 0; p < np; p++)
#pragma unroll
            for (int k = 0; k < V; k++) a.add(v[p][k], r);
        if constexpr (TOP) {
            asm volatile("" : "+v"(a.s), "+v"(a.t));  // the sums before the search
            // The bound is looked at after 1, 2, 4, ... calls, which every wave
            // of the block makes alike; a.m is the largest of a lane so far.
            if ((calls & (calls + 1)) == 0) {
                const float own = lp_bound(a.m, deep);
                if constexpr (NW == 1) top.at_least(own);
                else {
                    if (lane == 0) share[wave] = own;
                    // At the first call only: later values only raise the
                    // bound, and which of them a wave reads is of no
                    // consequence for the result.
                    if (!calls) __syncthreads();
                    float o[NW], bound = -INFINITY;
#pragma unroll
                    for (int w = 0; w < NW; w++) o[w] = share[w];
#pragma unroll
                    for (int w = 0; w < NW; w++) {
                        int reach = 0;
#pragma unroll
                        for (int z = 0; z < NW; z++) reach += o[z] >= o[w];
                        bound = fmaxf(bound, reach >= wide ? o[w] : -INFINITY);
                    }
                    top.at_least(bound);
                }
            }
            calls++;
            if (np == 1 && !in) {
                each[0] = __builtin_nanf("");
                raw[0] = lp_u32x4{~0u, ~0u, ~0u, ~0u};
            }
            // Every lane offers a pack's largest element, and while that is
            // good enough the next: the first of those equal to the maximum,
            // which is then put out of the way as a NaN.
#pragma unroll
            for (int p = 0; p < np; p++) {
                while (__any(each[p] >= top.worst)) {
                    // The pack is widened anew: its elements, kept over the
                    // search, would halve the waves of a SIMD.
                    asm volatile("" : "+v"(raw[p]));
                    float e[V];
                    int from = INT_MAX;
                    P::widen(raw[p], e);
#pragma unroll
                    for (int k = V - 1; k >= 0; k--) from = e[k] == each[p] ? k : from;
                    top.offer(each[p], from == INT_MAX ? INT_MAX : at + p * turn + from, g.top, lane);
                    P::drop(raw[p], from);
                    P::widen(raw[p], e);
                    each[p] = e[0];
#pragma unroll
                    for (int k = 1; k < V; k++) each[p] = fmaxf(each[p], e[k]);
                }
            }
        }
    };
    // The elements before the first boundary of 16 bytes and those behind the
    // last whole pack, one a thread: read first, added last.
    const int from = min(end, begin + (int)((0 - (uintptr_t)(x + begin)) % 16 / sizeof(typename P::S)));
    const int packs_end = from + (end - from) / V * V;
    const int odd = (int)threadIdx.x < from - begin ? begin + (int)threadIdx.x : packs_end - from + begin + (int)threadIdx.x;
    const float e = odd < end ? DType<DT>::to_c(x[odd]) : -INFINITY;
    const int mine = (int)threadIdx.x * V;
    int at = from;
    for (; at + UN * turn <= packs_end; at += UN * turn) take(at + mine, true, std::integral_constant<int, UN>{});
    for (; at < packs_end; at += turn) take(at + mine, at + mine < packs_end, std::integral_constant<int, 1>{});
    a.rise(e);
    if (odd < end) a.add(e, a.ref());
    if constexpr (TOP) {
        if (__any(e >= top.worst)) top.offer(e, odd < end ? odd : INT_MAX, g.top, lane);
    }
    a = lp_wave(a);
    if constexpr (NW > 1) {
        if (lane == 0) {
            box[wave][0] = a.m;
            box[wave][1] = a.s;
            box[wave][2] = a.t;
        }
        if constexpr (TOP) {
            top_v[wave][lane] = top.v;
            top_i[wave][lane] = top.i;
        }
        if constexpr (TOP) {
            if (wave == 0) {
                best_v[lane] = -INFINITY;
                best_i[lane] = INT_MAX;
            }
        }
        __syncthreads();
        if constexpr (TOP) {
            // an element's place among all waves' is its place in its own
            // list and the number of better ones in each other list, found
            // by halving
            int place = lane;
#pragma unroll
            for (int o = 1; o < NW; o++) {
                const int w = (wave + o) % NW;
                int low = 0, high = g.top;
                while (low < high) {
                    const int mid = (low + high) / 2;
                    if (LpTop::better(top_v[w][mid], top_i[w][mid], top.v, top.i)) low = mid + 1;
                    else high = mid;
                }
                place += low;
            }
            if (lane < g.top && place < g.top && top.i != INT_MAX) {
                best_v[place] = top.v;
                best_i[place] = top.i;
            }
            __syncthreads();
            top.v = best_v[lane];
            top.i = best_i[lane];
        }
        if (wave) return;
        for (int w = 1; w < NW; w++) a.join({box[w][0], box[w][1], box[w][2]});
    }
    if (g.splits == 1) {
        lp_finish(g, row, a, top, token, named, lane);
        return;
    }
    float *part = g.part + ((long long)row * g.splits + blockIdx.y) * (3 + 2 * g.top);
    if (lane == 0) {
        part[0] = a.m;
        part[1] = a.s;
        part[2] = a.t;
    }
    if (TOP && lane < g.top) {
        part[3 + lane] = top.v;
        part[3 + g.top + lane] = __builtin_bit_cast(float, top.i);
    }
}

// Joins the parts of a row, one wave a row.
template <int DT>
__global__ __launch_bounds__(64) void k_logprobs_join(LpArgs g)
{
    const int lane = threadIdx.x, row = blockIdx.x, width = 3 + 2 * g.top;
    const float *part = g.part + (long long)row * g.splits * width;
    bool named;
    const float token = lp_token<DT>(g, row, named);
    LpSum a;
    a.init();
    // Each part's list is in order.  With r = top / splits rounded up, j of
    // the parts' r-th elements have j r elements that are no smaller.
    const bool in = lane < g.splits;
    const float *list = part + lane * width + 3;
    const int r = (g.top + g.splits - 1) / g.splits;
    if (in) a = {part[lane * width], part[lane * width + 1], part[lane * width + 2]};
    float bound = -INFINITY, x = -INFINITY;
    int at = INT_MAX;
    if (in && g.top) {
        bound = list[r - 1];
        x = list[0];
        at = __builtin_bit_cast(int, list[g.top]);
    }
    a = lp_wave(a);
    LpTop top;
    top.init();
    if (g.top) top.at_least(lp_bound(bound, (g.top + r - 1) / r));
    for (int j = 0; j < g.top; j++) {
        // what follows in any list is no larger than its element j
        if (!__any(x >= top.worst)) break;
        float x2 = -INFINITY;
        int at2 = INT_MAX;
        if (in && j + 1 < g.top) {
            x2 = list[j + 1];
            at2 = __builtin_bit_cast(int, list[g.top + j + 1]);
        }
        top.offer(x, at, g.top, lane);
        x = x2;
        at = at2;
    }
    lp_finish(g, row, a, top, token, named, lane);
}

struct LpBwdArgs {
    const void *x;
    void *dx;
    long long stride;
    int rows, classes, per, top;
    const int32_t *tokens, *top_i;
    const float *stats, *entropy, *ga, *gh, *gu;
};

// One pass: x in, dx out (contiguous rows).  The few elements that carry a
// gradient of their own, the token's and the alternatives', are computed
// anew by single threads once the block's part of the row is written.
template <int DT, int NW>
__global__ __launch_bounds__(64 * NW) void k_logprobs_backward(LpBwdArgs g)
{
    using P = LpPack<DT>;
    using S = typename P::S;
    constexpr int V = P::V, UN = 4;
    const int row = blockIdx.x, lane = threadIdx.x & 63;
    const S *x = (const S *)g.x + (long long)row * g.stride;
    S *dx = (S *)g.dx + (long long)row * g.classes;
    const int begin = (int)min((long long)g.classes, (long long)g.per * blockIdx.y);
    const int end = (int)min((long long)g.classes, (long long)begin + g.per);

    int tok = g.tokens && g.ga ? g.tokens[row] : -1;
    const float m = g.stats[2 * (long long)row], log_s = g.stats[2 * (long long)row + 1];
    float own = tok >= 0 ? g.ga[row] : 0.0f;
    if (tok >= g.classes) own = __builtin_nanf("");  // as its log probability
    const float h = g.gh ? g.gh[row] : 0.0f;
    const float u = g.gu && lane < g.top ? g.gu[(long long)row * g.top + lane] : 0.0f;
    const int alt = g.gu && lane < g.top ? g.top_i[(long long)row * g.top + lane] : -1;
    const float all = own + (g.gu ? wave_all(alt >= 0 ? u : 0.0f, FAdd{}) : 0.0f);
    const bool none = m == -INFINITY && log_s == -INFINITY;
    const float r = m == -INFINITY ? 0.0f : m, base = h * (g.gh ? g.entropy[row] : 0.0f) + all;
    // -p (all + h (log p + H)); the logarithm is cut where p is 0
    auto common = [&](float e) {
        const float y = e - r - log_s, p = __builtin_amdgcn_exp2f(y * kLog2e);
        return -p * fmaf(h, fmaxf(y, -150.0f), base);
    };
    auto take = [&](int at, auto NP) {
        constexpr int np = decltype(NP)::value;
        lp_u32x4 raw[np];
        float v[np][V];
#pragma unroll
        for (int p = 0; p < np; p++) raw[p] = P::load(x + at + p * NW * 64 * V);
#pragma unroll
        for (int p = 0; p < np; p++) P::widen(raw[p], v[p]);
#pragma unroll
        for (int p = 0; p < np; p++) {
            union { lp_u32x4 raw; S s[V]; } o;
#pragma unroll
            for (int k = 0; k < V; k++) o.s[k] = DType<DT>::from_c(common(v[p][k]));
            __builtin_nontemporal_store(o.raw, (lp_u32x4 *)(dx + at + p * NW * 64 * V));
        }
    };
    const int turn = NW * 64 * V;
    int at = begin;
    if (none) {  // no distribution, no gradient
        for (int i = begin + (int)threadIdx.x; i < end; i += NW * 64) dx[i] = DType<DT>::from_c(0.0f);
        return;
    }
    for (; at + UN * turn <= end; at += UN * turn) take(at + (int)threadIdx.x * V, std::integral_constant<int, UN>{});
    for (; at + turn <= end; at += turn) take(at + (int)threadIdx.x * V, std::integral_constant<int, 1>{});
    for (int i = at + (int)threadIdx.x; i < end; i += NW * 64) dx[i] = DType<DT>::from_c(common(DType<DT>::to_c(x[i])));
    __syncthreads();  // the fence of this barrier orders the stores below behind those above
    if (threadIdx.x >= 64) return;
    // an alternative that is the token too adds both
    float mine = u;
    if (alt == tok) mine += own;
    if (alt >= begin && alt < end) dx[alt] = DType<DT>::from_c(common(DType<DT>::to_c(x[alt])) + mine);
    const bool listed = __any(alt >= 0 && alt == tok);
    if (lane == 0 && !listed && tok >= begin && tok < end)
        dx[tok] = DType<DT>::from_c(common(DType<DT>::to_c(x[tok])) + own);
}

template <int DT> static pt_status logprobs_typed(LpArgs g, hipStream_t s)
{
    // With few rows several blocks share one, 4096 elements each or more.
    const int most = std::min(64, (g.classes + 4095) / 4096);
    if (g.rows < 512 && most > 1) g.splits = std::min(most, (1024 + g.rows - 1) / g.rows);
    void *scratch = nullptr;
    if (g.splits > 1) {
        PT_TRY(scratch_alloc(&scratch, (size_t)g.rows * g.splits * (3 + 2 * (size_t)g.top) * sizeof(float), s));
        g.part = (float *)scratch;
    }
    const dim3 grid((unsigned)g.rows, (unsigned)g.splits);
    if (g.classes <= 2048) {
        if (g.top) k_logprobs<DT, 1, true><<<grid, 64, 0, s>>>(g);
        else k_logprobs<DT, 1, false><<<grid, 64, 0, s>>>(g);
    } else {
        if (g.top) k_logprobs<DT, 4, true><<<grid, 256, 0, s>>>(g);
        else k_logprobs<DT, 4, false><<<grid, 256, 0, s>>>(g);
    }
    if (g.splits > 1) k_logprobs_join<DT><<<(unsigned)g.rows, 64, 0, s>>>(g);
    const pt_status st = check_hip(hipGetLastError(), "log probabilities");
    if (scratch) scratch_free(scratch, s);
    return st;
}

template <int DT> static pt_status logprobs_backward_typed(LpBwdArgs g, hipStream_t s)
{
    const int most = std::min(64, (g.classes + 4095) / 4096);
    const int splits = g.rows < 512 && most > 1 ? std::min(most, (1024 + g.rows - 1) / g.rows) : 1;
    const int whole = 64 * LpPack<DT>::V;
    g.per = splits > 1 ? ((g.classes + splits - 1) / splits + whole - 1) / whole * whole : g.classes;
    const dim3 grid((unsigned)g.rows, (unsigned)splits);
    if (g.classes <= 2048) k_logprobs_backward<DT, 1><<<grid, 64, 0, s>>>(g);
    else k_logprobs_backward<DT, 4><<<grid, 256, 0, s>>>(g);
    return check_hip(hipGetLastError(), "log probability gradient");
}

// A launch counts its threads in 32 bits: this many rows at once.
constexpr size_t kLpRows = 1u << 22;

static pt_status logprobs_check(int dtype, size_t rows, size_t classes, size_t row_stride, int top)
{
    if (dtype != PT_FLOAT32 && dtype != PT_FLOAT16 && dtype != PT_BFLOAT16)
        return fail(PT_ERR_INVALID, "log probabilities require float32, float16 or bfloat16 scores");
    if (rows > (size_t)INT_MAX || classes > (size_t)INT_MAX - 65536)
        return fail(PT_ERR_INVALID, "log probabilities count rows and classes in 32 bits");
    if (rows && !classes) return fail(PT_ERR_INVALID, "log probabilities need at least one class");
    if (rows > 1 && row_stride < classes) return fail(PT_ERR_INVALID, "log probability rows overlap");
    if (top < 0 || top > 64 || (rows && (size_t)top > classes))
        return fail(PT_ERR_INVALID, "log probabilities list 0 to 64 alternatives, and no more than the classes");
    return PT_OK;
}

}  // namespace pt

using namespace pt;

extern "C" {

pt_status pt_logprobs(const void *logits, int dtype, size_t rows, size_t classes, size_t row_stride,
                      const int32_t *tokens, int top, float *logprob, float *entropy, float *stats, float *top_logprob,
                      int32_t *top_index, pt_stream_t stream)
{
    PT_TRY(logprobs_check(dtype, rows, classes, row_stride, top));
    if (rows && (!logits || (logprob && !tokens))) return fail(PT_ERR_INVALID, "log probabilities miss an operand");
    PT_TRY(ensure_init());
    if (!rows) return PT_OK;
    counters().fused_row_calls++;
    hipStream_t s = stream_of(stream);
    for (size_t from = 0; from < rows; from += kLpRows) {
        auto at = [&](auto *p, size_t width) { return p ? p + from * width : nullptr; };
        const LpArgs g = {(const char *)logits + from * row_stride * dtype_size(dtype), (long long)row_stride,
                          (int)std::min(rows - from, kLpRows), (int)classes, 1, top, at(tokens, 1), at(logprob, 1),
                          at(entropy, 1), at(stats, 2), at(top_logprob, top), at(top_index, top), nullptr};
        switch (dtype) {
        case PT_FLOAT32: PT_TRY(logprobs_typed<PT_FLOAT32>(g, s)); break;
        case PT_FLOAT16: PT_TRY(logprobs_typed<PT_FLOAT16>(g, s)); break;
        default: PT_TRY(logprobs_typed<PT_BFLOAT16>(g, s));
        }
    }
    return PT_OK;
}

pt_status pt_logprobs_backward(const void *logits, int dtype, size_t rows, size_t classes, size_t row_stride,
                               const int32_t *tokens, int top, const int32_t *top_index, const float *stats,
                               const float *entropy, const float *grad_logprob, const float *grad_entropy,
                               const float *grad_top, void *dlogits, pt_stream_t stream)
{
    PT_TRY(logprobs_check(dtype, rows, classes, row_stride, top));
    if (rows && (!logits || !stats || !dlogits || (grad_logprob && !tokens) || (grad_entropy && !entropy) ||
                 (grad_top && top && !top_index)))
        return fail(PT_ERR_INVALID, "log probability gradient misses an operand");
    PT_TRY(ensure_init());
    if (!rows) return PT_OK;
    counters().fused_row_calls++;
    hipStream_t s = stream_of(stream);
    const size_t es = dtype_size(dtype);
    for (size_t from = 0; from < rows; from += kLpRows) {
        auto at = [&](auto *p, size_t width) { return p ? p + from * width : nullptr; };
        const LpBwdArgs g = {(const char *)logits + from * row_stride * es, (char *)dlogits + from * classes * es,
                             (long long)row_stride, (int)std::min(rows - from, kLpRows), (int)classes, 0, top, at(tokens, 1),
                             at(top_index, top), at(stats, 2), at(entropy, 1), at(grad_logprob, 1), at(grad_entropy, 1),
                             top ? at(grad_top, top) : nullptr};
        switch (dtype) {
        case PT_FLOAT32: PT_TRY(logprobs_backward_typed<PT_FLOAT32>(g, s)); break;
        case PT_FLOAT16: PT_TRY(logprobs_backward_typed<PT_FLOAT16>(g, s)); break;
        default: PT_TRY(logprobs_backward_typed<PT_BFLOAT16>(g, s));
        }
    }
    return PT_OK;
}

}  // extern "C"
