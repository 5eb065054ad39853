// Rotation of queries and keys by their positions, with the norm of each head
// in the same pass, for gfx950.  A head x of `size` elements at position t:
//   n = x, or n_j = x_j r w_j with r = 1 / sqrt(mean(x^2) + eps)
//   (y_p, y_q) = (c n_p - s n_q, s n_p + c n_q),  c = m cos(t f_i), s = m sin(t f_i)
// for the pairs (p, q) = (i, i + part / 2) or (2i, 2i + 1) of its first
// `part` elements; the others pass.  Gradient: dn is the upstream gradient
// rotated back; dx = dn, or with h = dn w and u = x r
//   dw = sum dn u,   dx = r (h - u mean(h u)).
// HBM-bound: a head is read once (with its upstream gradient) and written
// once.  A lane's unit of work is 2 V elements, V a 16-byte pack: V pairs, or
// 2 V elements that pass; a head takes the power of two of lanes that holds
// its units, so its sum of squares is a few exchanges inside a wave.  Waves
// work on their own: a wave takes one token and walks its heads, the next
// ones on their way while it turns these.  It computes the token's angles
// once for all of them, a pair or two a lane, and hands them round through
// its own part of LDS without a barrier: as turns, reduced in double before
// they are rounded (positions reach 2^31).  One cosine and sine per element
// would cost more than the memory.  Blocks with barriers, a head to a group of
// waves, took twice as long.
// Measured, bfloat16, 8192 tokens, 32 and 8 heads of 128 with norms: forward
// 36 us (4.7 TB/s; a large copy 5.0), gradients of the 32 heads 43-45 us (4.5
// TB/s) and of the 8 17-18 us, each scale's sum 4.8 us; one token for each of
// 32 texts 4.5 us.
#include "pt_common.h"

#include <algorithm>
#include <math.h>

namespace pt {

constexpr int kRotWaves = 4;
constexpr int kRotBlocks = 2048;

struct RotSide {
    const void *x;      // null in a backward pass without a norm
    const void *scale;  // null: no norm
    const void *g;      // upstream gradient, contiguous (backward pass)
    void *y;            // result, contiguous
    float *partial;     // [block][size] of the scale's gradient, or null
    long long st[3];    // sequence, token, head
    int heads;
};

struct RotArgs {
    RotSide side[2];
    const double *turns;        // frequencies / 2 pi
    const int32_t *positions;   // null: a sequence's tokens from 0 on
    long long pst[2];           // sequence, token
    unsigned tokens, rows;      // of a sequence, of all
    int size, part, lanes_log2;
    int passes;                 // a wave's turns over 64 >> lanes_log2 heads of a token
    float magnitude, eps;
};

// Unit u of a head: elements at[0] .. +V - 1 and at[1] .. +V - 1, of which
// `live` of each belong to it, the first `turned` of V pairs among them.
// Pairs (2i, 2i + 1): 2 V elements in a row, the end of the turned part
// inside of one.  Pairs (i, i + part / 2): V in both halves of that part, and
// units of their own behind it.
struct RotUnit {
    int at[2], live[2], turned;
};

// V of a kernel: 16 bytes, and 8 in a backward pass in 16 bits, whose values
// then take 100 registers instead of 160 (8192 tokens of 32 heads of 128: 43
// against 50 us; the forward pass 36 us with 16 bytes, 43 with 8)
__host__ __device__ constexpr int rot_width(int dtype, bool back) { return dtype == PT_FLOAT32 || back ? 4 : 8; }
__host__ __device__ inline int rot_units(int size, int part, bool paired, int v)
{
    return paired ? (size + 2 * v - 1) / (2 * v) : (part / 2 + v - 1) / v + (size - part + 2 * v - 1) / (2 * v);
}

template <int V, bool PAIRED>
__device__ __forceinline__ RotUnit rot_unit(const RotArgs &a, int u)
{
    const int pairs = a.part / 2, units = (pairs + V - 1) / V;
    RotUnit r;
    r.turned = max(0, min(V, pairs - u * V));
    const bool halves = !PAIRED && r.turned;
    const int base = PAIRED ? 2 * V * u : halves ? V * u : a.part + (u - units) * 2 * V;
    r.at[0] = base;
    r.at[1] = halves ? pairs + base : base + V;
    r.live[0] = halves ? r.turned : max(0, min(V, a.size - base));
    r.live[1] = halves ? r.turned : max(0, min(V, a.size - base - V));
    return r;
}

// What a unit's elements are in memory, in whole registers.
template <int DT, int V> struct RotRaw {
    static constexpr int N = V * (int)sizeof(typename DType<DT>::S) / 4;
    typedef unsigned words __attribute__((ext_vector_type(N), aligned(1)));
    words q[2];
};

// (16 bytes load and store at any element boundary)
template <int DT, int V>
__device__ __forceinline__ void rot_read(const void *base, long long off, const RotUnit &r, RotRaw<DT, V> &raw)
{
    using S = typename DType<DT>::S;
    using Words = typename RotRaw<DT, V>::words;
    const S *p = (const S *)base + off;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (r.live[h] == V) {
            raw.q[h] = *(const Words *)(p + r.at[h]);
        } else {
            union { Words q; S s[V]; } u;
#pragma unroll
            for (int i = 0; i < V; i++) u.s[i] = i < r.live[h] ? p[r.at[h] + i] : (S)0;
            raw.q[h] = u.q;
        }
    }
}
template <int DT, int V>
__device__ __forceinline__ void rot_values(const RotRaw<DT, V> &raw, float (&v)[2 * V])
{
    constexpr bool LOW = DT != PT_FLOAT32;
#pragma unroll
    for (int i = 0; i < 2 * V; i++) {
        const unsigned word = raw.q[i / V][LOW ? (i % V) / 2 : i % V];
        if constexpr (!LOW) v[i] = __uint_as_float(word);
        else if constexpr (DT == PT_BFLOAT16) v[i] = __uint_as_float(i & 1 ? word & 0xffff0000u : word << 16);
        else v[i] = f16_to_float((uint16_t)(i & 1 ? word >> 16 : word));
    }
}
template <int DT, int V>
__device__ __forceinline__ void rot_write(void *base, long long off, const RotUnit &r, const float (&v)[2 * V])
{
    using S = typename DType<DT>::S;
    using Words = typename RotRaw<DT, V>::words;
    S *p = (S *)base + off;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (r.live[h] == V) {
            Words q;
#pragma unroll
            for (int i = 0; i < RotRaw<DT, V>::N; i++) {
                if constexpr (DT == PT_FLOAT32) q[i] = __float_as_uint(v[h * V + i]);
                else q[i] = pack_low<DT>(v[h * V + 2 * i], v[h * V + 2 * i + 1]);
            }
            __builtin_nontemporal_store(q, (Words *)(p + r.at[h]));
        } else
#pragma unroll
            for (int i = 0; i < V; i++)
                if (i < r.live[h]) p[r.at[h] + i] = DType<DT>::from_c(v[h * V + i]);
    }
}

// the first n pairs of v turned by their angles, backwards with sign -1
template <int V, bool PAIRED>
__device__ __forceinline__ void rot_turn(const float2 (&angle)[V], int n, float sign, float (&v)[2 * V])
{
    if (!n) return;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int p = PAIRED ? 2 * i : i, q = PAIRED ? 2 * i + 1 : V + i;
        const float x = v[p], y = v[q], s = sign * angle[i].y;
        const float a = x * angle[i].x - y * s, b = x * s + y * angle[i].x;
        v[p] = PAIRED && i >= n ? x : a;  // (in halves what is past the end is not stored)
        v[q] = PAIRED && i >= n ? y : b;
    }
}

// the sum over the 2^log2 lanes that share a head (log2 is uniform): up to
// 16 lanes by DPP (pairs, quads, mirrored halves of a row), without LDS
__device__ __forceinline__ float rot_sum(float v, int log2)
{
    auto with = [](float x, auto CTRL) {
        return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(CTRL)::value, 0xF, 0xF, false));
    };
    if (log2 > 0) v = with(v, std::integral_constant<int, 0xB1>{});
    if (log2 > 1) v = with(v, std::integral_constant<int, 0x4E>{});
    if (log2 > 2) v = with(v, std::integral_constant<int, 0x141>{});
    if (log2 > 3) v = with(v, std::integral_constant<int, 0x140>{});
    if (log2 > 4) v += __shfl_xor(v, 16, PT_WAVE);
    if (log2 > 5) v += __shfl_xor(v, 32, PT_WAVE);
    return v;
}

// Forward: the heads of both sides count through.  Backward: blockIdx.y is
// the side, so that a lane's part of the scale's gradient stays in registers
// over all the tokens that its wave takes.
// MANY: a token's heads fill half of a wave at most, so it takes as many tokens
// at once as do fill it (`groups`); each lane finds its own token's.  2 heads of
// 32 in bfloat16 3.5 TB/s instead of 0.6, 8 heads of 32 4.4 instead of 2.2.
template <int DT, int GDT, bool PAIRED, bool BACK, bool MANY>
__global__ __launch_bounds__(64 * kRotWaves) void k_rotary(RotArgs a)
{
    constexpr int V = rot_width(DT, BACK);
    using Raw = RotRaw<DT, V>;
    __shared__ float2 tables[kRotWaves][MANY ? 64 * V : 128];
    __shared__ float sums[BACK ? kRotWaves : 1][BACK ? 2 * V : 1][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int log2 = a.lanes_log2, u = lane & ((1 << log2) - 1), slot = lane >> log2, slots = 64 >> log2;
    const int pairs = a.part / 2;
    const RotSide &s0 = a.side[BACK ? blockIdx.y : 0], &s1 = a.side[1];
    const unsigned heads = BACK ? s0.heads : s0.heads + s1.heads;
    const unsigned units = (heads + slots * a.passes - 1) / (slots * a.passes);  // of a token
    // a lane's token of those that a wave takes, and its head on the first pass
    const unsigned groups = MANY ? slots / heads : 1, group = MANY ? slot / heads : 0;
    const unsigned head0 = MANY ? (group < groups ? slot - group * heads : heads) : slot;
    const RotUnit unit = rot_unit<V, PAIRED>(a, u);
    const float inv_n = 1.0f / (float)a.size;
    float2 *table = tables[wave];
    // the token and the first head of a wave's turn; rows times units are below 2^48
    struct Turn {
        unsigned row, seq, t, first;
        long long pos;
    };
    const unsigned long long total = ((unsigned long long)a.rows + groups - 1) / groups * units;
    const unsigned long long step = (unsigned long long)gridDim.x * kRotWaves;
    auto place = [&](unsigned row, Turn &n) {
        n.row = row;
        n.seq = a.tokens == a.rows ? 0 : row / a.tokens;
        n.t = row - n.seq * a.tokens;
        n.pos = a.positions ? (long long)a.positions[n.seq * a.pst[0] + n.t * a.pst[1]] : (long long)n.t;
    };
    auto turn_of = [&](unsigned long long at) {
        Turn n;
        const unsigned turn = units == 1 ? (unsigned)at : (unsigned)(at / units);
        n.first = (unsigned)(at - (unsigned long long)turn * units) * a.passes * slots;
        if constexpr (MANY) {  // (past the last token: that one again, and no head)
            const unsigned long long row = (unsigned long long)turn * groups + group;
            n.first = row < a.rows ? 0 : heads;
            place((unsigned)min(row, (unsigned long long)a.rows - 1), n);
        } else {
            place(turn, n);
        }
        return n;
    };
    auto fetch = [&](const Turn &n, unsigned h, Raw &x, RotRaw<GDT, V> &g) {
        if (h >= heads) return;
        const bool key = !BACK && h >= (unsigned)s0.heads;
        const RotSide &s = key ? s1 : s0;
        const unsigned head = key ? h - s0.heads : h;
        if (!BACK || s.scale) rot_read<DT, V>(s.x, n.seq * s.st[0] + n.t * s.st[1] + head * s.st[2], unit, x);
        if constexpr (BACK) rot_read<GDT, V>(s.g, ((long long)n.row * s.heads + head) * a.size, unit, g);
    };
    unsigned long long at = (unsigned long long)blockIdx.x * kRotWaves + wave;
    Raw x, xn, w0, w1;
    RotRaw<GDT, V> g, gn;
    Turn now = {}, next = {};
    if (at < total) {
        now = turn_of(at);
        fetch(now, now.first + head0, x, g);
    }
    if (s0.scale) rot_read<DT, V>(s0.scale, 0, unit, w0);
    if (!BACK && s1.scale) rot_read<DT, V>(s1.scale, 0, unit, w1);
    const double turns0 = a.turns[min(lane, pairs - 1)], turns1 = a.turns[min(lane + 64, pairs - 1)];
    float dw[2 * V];
#pragma unroll
    for (int i = 0; i < 2 * V; i++) dw[i] = 0.0f;
    for (; at < total; at += step) {
        const bool more = at + step < total;
        if (more) next = turn_of(at + step);
        for (int f = lane; f < (int)groups * pairs; f += 64) {
            long long pos = now.pos;
            double each = f < 64 ? turns0 : turns1;
            if constexpr (MANY) {
                const int of = f / pairs;
                Turn n;
                place((unsigned)min((unsigned long long)(at * groups + of), (unsigned long long)a.rows - 1), n);
                pos = n.pos;
                each = a.turns[f - of * pairs];
            }
            // the fraction of a turn in two floats: the second corrects the first's cosine and sine
            double turns = (double)pos * each;
            turns -= rint(turns);
            const float hi = (float)turns, lo = (float)(turns - (double)hi) * 6.28318531f;
            float sn, cs;
            sincospif(2.0f * hi, &sn, &cs);
            table[f] = make_float2((cs - lo * sn) * a.magnitude, (sn + lo * cs) * a.magnitude);
        }
        // the table is this wave's own: its LDS accesses stay in order
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        float2 angle[V];
#pragma unroll
        for (int i = 0; i < V; i++) angle[i] = table[(MANY ? min(group, groups - 1) * pairs : 0) + min(u * V + i, pairs - 1)];
        __builtin_amdgcn_wave_barrier();
        for (int p = 0; p < a.passes; p++) {
            const unsigned h = now.first + p * slots + head0;
            if (p + 1 < a.passes) fetch(now, h + slots, xn, gn);
            else if (more) fetch(next, next.first + head0, xn, gn);
            if (h < heads) {  // (whole groups of lanes, so a head's sum has all its lanes)
                const bool key = !BACK && h >= (unsigned)s0.heads;
                const RotSide &s = key ? s1 : s0;
                const unsigned head = key ? h - s0.heads : h;
                const long long to = ((long long)now.row * s.heads + head) * a.size;
                float v[2 * V], w[2 * V];
                rot_values<DT, V>(x, v);
                if constexpr (!BACK) {
                    if (s.scale) {
                        rot_values<DT, V>(key ? w1 : w0, w);
                        float q = 0.0f;
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) q = fmaf(v[i], v[i], q);
                        const float r = 1.0f / sqrtf(rot_sum(q, log2) * inv_n + a.eps);
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) v[i] = v[i] * r * w[i];
                    }
                    rot_turn<V, PAIRED>(angle, unit.turned, 1.0f, v);
                    rot_write<DT, V>(s.y, to, unit, v);
                } else {
                    float d[2 * V];
                    rot_values<GDT, V>(g, d);
                    rot_turn<V, PAIRED>(angle, unit.turned, -1.0f, d);
                    if (s.scale) {
                        rot_values<DT, V>(w0, w);
                        float q = 0.0f, b = 0.0f;
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) {
                            q = fmaf(v[i], v[i], q);
                            b = fmaf(d[i] * w[i], v[i], b);
                        }
                        const float r = 1.0f / sqrtf(rot_sum(q, log2) * inv_n + a.eps);
                        b = rot_sum(b, log2) * inv_n * r;
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) {
                            const float n = v[i] * r;
                            dw[i] = fmaf(d[i], n, dw[i]);
                            d[i] = r * (d[i] * w[i] - n * b);
                        }
                    }
                    if (s.y) rot_write<DT, V>(s.y, to, unit, d);
                }
            }
            x = xn;
            if constexpr (BACK) g = gn;
        }
        now = next;
    }
    if constexpr (BACK) {
        if (!s0.partial) return;
#pragma unroll
        for (int i = 0; i < 2 * V; i++) {
            for (int m = 1 << log2; m < 64; m <<= 1) dw[i] += __shfl_xor(dw[i], m, PT_WAVE);
            sums[wave][i][lane] = dw[i];
        }
        __syncthreads();
        if (wave || slot) return;
#pragma unroll
        for (int i = 0; i < 2 * V; i++) {
            float t = dw[i];
            for (int o = 1; o < kRotWaves; o++) t += sums[o][i][lane];
            if (i % V < unit.live[i / V]) s0.partial[(long long)blockIdx.x * a.size + unit.at[i / V] + i % V] = t;
        }
    }
}

// The scale's gradient from the blocks' partial rows, in a fixed order: a
// wave adds four columns, its lanes every 16th row.
template <int DT>
__global__ __launch_bounds__(64) void k_rotary_scale(RotArgs a, int parts, void *d0, void *d1)
{
    const int c = (int)blockIdx.x * 4 + (threadIdx.x & 3);
    void *out = blockIdx.y ? d1 : d0;
    const float *p = a.side[blockIdx.y].partial;
    if (!out) return;  // whole block
    float t = 0.0f;
    if (c < a.size)
#pragma unroll 8
        for (int r = threadIdx.x >> 2; r < parts; r += 16) t += p[(long long)r * a.size + c];
    for (int m = 4; m < 64; m <<= 1) t += __shfl_xor(t, m, PT_WAVE);
    if (threadIdx.x < 4 && c < a.size) ((typename DType<DT>::S *)out)[c] = DType<DT>::from_c(t);
}

template <int DT, int GDT, bool BACK>
static void launch_rotary_as(const RotArgs &a, bool interleaved, bool many, dim3 grid, hipStream_t s)
{
    if (many) {
        if (interleaved) k_rotary<DT, GDT, true, BACK, true><<<grid, 64 * kRotWaves, 0, s>>>(a);
        else k_rotary<DT, GDT, false, BACK, true><<<grid, 64 * kRotWaves, 0, s>>>(a);
    } else {
        if (interleaved) k_rotary<DT, GDT, true, BACK, false><<<grid, 64 * kRotWaves, 0, s>>>(a);
        else k_rotary<DT, GDT, false, BACK, false><<<grid, 64 * kRotWaves, 0, s>>>(a);
    }
}
template <int DT, int GDT>
static void launch_rotary(const RotArgs &a, bool interleaved, bool back, bool many, dim3 grid, hipStream_t s)
{
    if (back) return launch_rotary_as<DT, GDT, true>(a, interleaved, many, grid, s);
    if constexpr (DT == GDT) launch_rotary_as<DT, DT, false>(a, interleaved, many, grid, s);
}

// How the heads go to waves: a wave's passes over a token's heads, as many as
// leave 8192 waves (two for each slot of the GPU at a register count of 128).
// many: several tokens fit a wave, and there are so many of them that it pays
// (one head of 128 in bfloat16: 2048 tokens 4.6 us alone, 6.4 together; 4096
// 6.0 and 6.5, 2 heads of 64 6.1 and 5.3; 16384 14 and 7).
static unsigned rotary_blocks(RotArgs &a, int dtype, bool paired, bool back, int heads, long long most, bool &many)
{
    const int units = rot_units(a.size, a.part, paired, rot_width(dtype, back));
    a.lanes_log2 = 0;
    while (1 << a.lanes_log2 < units) a.lanes_log2++;  // (at most 64: heads have at most 256 elements)
    const int all = (heads + (64 >> a.lanes_log2) - 1) >> (6 - a.lanes_log2);
    a.passes = (int)std::max<long long>(1, std::min<long long>(all, (long long)a.rows * all / 8192));
    const int groups = (64 >> a.lanes_log2) / heads;  // (of the side with more heads)
    many = groups > 1 && a.rows >= 4096;
    const long long waves = many ? ((long long)a.rows + groups - 1) / groups : (long long)a.rows * ((all + a.passes - 1) / a.passes);
    // (in rounds of equal length)
    const long long blocks = (waves + kRotWaves - 1) / kRotWaves, rounds = (blocks + most - 1) / most;
    return (unsigned)((blocks + rounds - 1) / rounds);
}

static pt_status rotary_args(const pt_rotary_desc *d, RotArgs &a)
{
    if (!d) return fail(PT_ERR_INVALID, "rotary description missing");
    if (d->dtype != PT_FLOAT32 && d->dtype != PT_FLOAT16 && d->dtype != PT_BFLOAT16)
        return fail(PT_ERR_INVALID, "rotary takes float32, float16 or bfloat16 heads");
    if (d->sequences < 0 || d->tokens < 0 || d->heads[0] < 0 || d->heads[1] < 0)
        return fail(PT_ERR_INVALID, "rotary counts must not be negative");
    if (d->size < 1 || d->part < 2 || d->part % 2 || d->part > d->size)
        return fail(PT_ERR_INVALID, "rotary turns an even number of a head's elements");
    if (d->size > 256) return fail(PT_ERR_UNSUPPORTED, "rotary heads have at most 256 elements");
    if (!d->turns) return fail(PT_ERR_INVALID, "rotary frequencies missing");
    if (!isfinite(d->magnitude) || !isfinite((float)d->magnitude))
        return fail(PT_ERR_INVALID, "rotary magnitude must be finite");
    if (!(d->epsilon > 0.0) || !isfinite((float)d->epsilon) || (float)d->epsilon <= 0.0f)
        return fail(PT_ERR_INVALID, "rotary epsilon must be finite and greater than zero");
    const long long rows = (long long)d->sequences * d->tokens;
    if (rows > INT32_MAX || d->heads[0] > 65536 || d->heads[1] > 65536)
        return fail(PT_ERR_INVALID, "rotary has too many tokens or heads");
    a.turns = d->turns;
    a.positions = d->positions;
    a.pst[0] = (long long)d->position_strides[0];
    a.pst[1] = (long long)d->position_strides[1];
    a.tokens = (unsigned)std::max(1, d->tokens);
    a.rows = (unsigned)rows;
    a.size = d->size;
    a.part = d->part;
    a.magnitude = (float)d->magnitude;
    a.eps = (float)d->epsilon;
    for (int i = 0; i < 2; i++) {
        a.side[i].heads = d->heads[i];
        for (int k = 0; k < 3; k++) a.side[i].st[k] = (long long)d->strides[i][k];
    }
    return PT_OK;
}

}  // namespace pt

using namespace pt;

extern "C" {

pt_status pt_rotary(const pt_rotary_desc *d, const void *const *x, const void *const *scale, void *const *y,
                    pt_stream_t stream)
{
    RotArgs a = {};
    PT_TRY(rotary_args(d, a));
    if (!x || !y) return fail(PT_ERR_INVALID, "rotary misses an operand");
    int sides = 0;
    for (int i = 0; i < 2; i++) {
        RotSide &s = a.side[i];
        if (!s.heads || !a.rows) continue;
        if (!x[i] || !y[i]) return fail(PT_ERR_INVALID, "rotary misses an operand");
        s.x = x[i];
        s.y = y[i];
        s.scale = scale ? scale[i] : nullptr;
        if (sides != i) std::swap(a.side[0], a.side[1]);
        sides++;
    }
    PT_TRY(ensure_init());
    if (!sides) return PT_OK;
    hipStream_t s = stream_of(stream);
    if (sides == 1) a.side[1].heads = 0;
    bool many;
    const unsigned blocks = rotary_blocks(a, d->dtype, d->interleaved, false, a.side[0].heads + a.side[1].heads, kRotBlocks, many);
    if (d->dtype == PT_FLOAT32) launch_rotary<PT_FLOAT32, PT_FLOAT32>(a, d->interleaved, false, many, blocks, s);
    else if (d->dtype == PT_FLOAT16) launch_rotary<PT_FLOAT16, PT_FLOAT16>(a, d->interleaved, false, many, blocks, s);
    else launch_rotary<PT_BFLOAT16, PT_BFLOAT16>(a, d->interleaved, false, many, blocks, s);
    return check_hip(hipGetLastError(), "rotary");
}

pt_status pt_rotary_backward(const pt_rotary_desc *d, const void *const *x, const void *const *scale,
                             const void *const *grad, int grad_dtype, void *const *dx, void *const *dscale,
                             pt_stream_t stream)
{
    RotArgs a = {};
    PT_TRY(rotary_args(d, a));
    if (grad_dtype != d->dtype && grad_dtype != PT_FLOAT32)
        return fail(PT_ERR_INVALID, "rotary's upstream gradient must be float32 or of the heads' dtype");
    if (!grad || !dx) return fail(PT_ERR_INVALID, "rotary gradient misses an operand");
    void *ds[2] = {nullptr, nullptr};
    int sides = 0;
    bool partial = false;
    for (int i = 0; i < 2; i++) {
        RotSide &s = a.side[i];
        s.scale = scale ? scale[i] : nullptr;
        void *to = s.scale && dscale ? dscale[i] : nullptr;
        if (!s.heads || !a.rows) {
            // no head adds anything: the scale's gradient is zeros
            const pt_scalar_t zero = {{0.0}, d->dtype};
            if (to) PT_TRY(pt_fill(to, d->dtype, (size_t)d->size, &zero, stream));
            continue;
        }
        if (!grad[i] || (!dx[i] && !to) || (s.scale && (!x || !x[i])))
            return fail(PT_ERR_INVALID, "rotary gradient misses an operand");
        s.x = s.scale ? x[i] : nullptr;
        s.g = grad[i];
        s.y = dx[i];
        ds[sides] = to;
        partial = partial || to;
        if (sides != i) std::swap(a.side[0], a.side[1]);
        sides++;
    }
    PT_TRY(ensure_init());
    if (!sides) return PT_OK;
    hipStream_t s = stream_of(stream);
    // a partial row a block: four blocks a CU walk the tokens
    bool many;
    const unsigned blocks = rotary_blocks(a, d->dtype, d->interleaved, true, std::max(a.side[0].heads, sides > 1 ? a.side[1].heads : 0),
                                          partial ? kRotBlocks / 2 : kRotBlocks, many);
    void *scratch = nullptr;
    if (partial) {
        PT_TRY(scratch_alloc(&scratch, (size_t)blocks * 2 * a.size * sizeof(float), s));
        for (int i = 0; i < sides; i++)
            if (ds[i]) a.side[i].partial = (float *)scratch + (size_t)i * blocks * a.size;
    }
    const bool same = grad_dtype == d->dtype;
    if (d->dtype == PT_FLOAT32) launch_rotary<PT_FLOAT32, PT_FLOAT32>(a, d->interleaved, true, many, dim3(blocks, sides), s);
    else if (d->dtype == PT_FLOAT16) {
        if (same) launch_rotary<PT_FLOAT16, PT_FLOAT16>(a, d->interleaved, true, many, dim3(blocks, sides), s);
        else launch_rotary<PT_FLOAT16, PT_FLOAT32>(a, d->interleaved, true, many, dim3(blocks, sides), s);
    } else {
        if (same) launch_rotary<PT_BFLOAT16, PT_BFLOAT16>(a, d->interleaved, true, many, dim3(blocks, sides), s);
        else launch_rotary<PT_BFLOAT16, PT_FLOAT32>(a, d->interleaved, true, many, dim3(blocks, sides), s);
    }
    if (partial) {
        const dim3 grid((a.size + 3) / 4, sides);
        if (d->dtype == PT_FLOAT32) k_rotary_scale<PT_FLOAT32><<<grid, 64, 0, s>>>(a, (int)blocks, ds[0], ds[1]);
        else if (d->dtype == PT_FLOAT16) k_rotary_scale<PT_FLOAT16><<<grid, 64, 0, s>>>(a, (int)blocks, ds[0], ds[1]);
        else k_rotary_scale<PT_BFLOAT16><<<grid, 64, 0, s>>>(a, (int)blocks, ds[0], ds[1]);
    }
    const pt_status st = check_hip(hipGetLastError(), "rotary gradient");
    if (scratch) scratch_free(scratch, s);
    return st;
}

}  // extern "C"
