// Rotation of queries and keys by their positions, with the norm of each head
// in the same pass, for gfx950.  A head x of `size` elements at position t:
//   n = x, or n_j = x_j r w_j with r = 1 / sqrt(mean(x^2) + eps)
//   (y_p, y_q) = (c n_p - s n_q, s n_p + c n_q),  c = m cos(t f_i), s = m sin(t f_i)
// for the pairs (p, q) = (i, i + part / 2) or (2i, 2i + 1) of its first
// `part` elements; the others pass.  Gradient: dn is the upstream gradient
// rotated back; dx = dn, or with h = dn w and u = x r
//   dw = sum dn u,   dx = r (h - u mean(h u)).
// HBM-bound: a head is read once (with its upstream gradient) and written
// once.  A unit of work is 2 V elements (V a 16-byte pack where the pairs
// allow it): V pairs, or 2 V elements that pass; a head takes the power of
// two of lanes that holds its units, so its sum of squares is a few
// exchanges inside a wave.  The angles of a block's tokens are computed once
// into LDS, in double (turns, reduced before they are rounded: positions
// reach 2^31), while the first heads are on their way, and serve all heads:
// one cosine and sine per element would cost more than the memory.
#include "pt_common.h"

#include <algorithm>
#include <math.h>

namespace pt {

constexpr int kRotThreads = 256;
constexpr int kRotTable = 256;  // pairs whose cosines and sines a block holds

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
    int group;                  // tokens that a block takes at a time
    float magnitude, eps;
};

template <int DT, int V>
__device__ __forceinline__ void rot_load(const typename DType<DT>::S *p, float *v)
{
    using S = typename DType<DT>::S;
    typedef S vec __attribute__((ext_vector_type(V), aligned(sizeof(S))));
    if constexpr (V == 1) v[0] = DType<DT>::to_c(*p);
    else {
        const vec r = *(const vec *)p;
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = DType<DT>::to_c(r[i]);
    }
}

template <int DT, int V>
__device__ __forceinline__ void rot_store(typename DType<DT>::S *p, const float *v)
{
    using S = typename DType<DT>::S;
    typedef S vec __attribute__((ext_vector_type(V), aligned(sizeof(S))));
    if constexpr (V == 1) *p = DType<DT>::from_c(v[0]);
    else {
        vec r;
#pragma unroll
        for (int i = 0; i < V; i++) r[i] = DType<DT>::from_c(v[i]);
        *(vec *)p = r;
    }
}

// Unit u of a head: elements at[0] .. +V - 1 and at[1] .. +V - 1, `live` of
// the 2 V in order that belong to the head, rotated where u < part / 2 / V.
struct RotUnit {
    int at[2];
    int live;
    bool turned;
};

template <int V, bool PAIRED>
__device__ __forceinline__ RotUnit rot_unit(const RotArgs &a, int u)
{
    const int pairs = a.part / 2, units = pairs / V;
    RotUnit r;
    r.turned = u < units;
    r.live = 2 * V;
    if (r.turned) {
        r.at[0] = PAIRED ? 2 * V * u : V * u;
        r.at[1] = PAIRED ? 2 * V * u + V : pairs + V * u;
    } else {
        r.at[0] = a.part + (u - units) * 2 * V;
        r.at[1] = r.at[0] + V;
        r.live = max(0, min(2 * V, a.size - r.at[0]));
    }
    return r;
}

template <int DT, int V>
__device__ __forceinline__ void rot_read(const void *base, long long off, const RotUnit &r, float (&v)[2 * V])
{
    using S = typename DType<DT>::S;
    const S *p = (const S *)base + off;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (r.live >= (h + 1) * V) rot_load<DT, V>(p + r.at[h], v + h * V);
        else
#pragma unroll
            for (int i = 0; i < V; i++) v[h * V + i] = h * V + i < r.live ? DType<DT>::to_c(p[r.at[h] + i]) : 0.0f;
    }
}

template <int DT, int V>
__device__ __forceinline__ void rot_write(void *base, long long off, const RotUnit &r, const float (&v)[2 * V])
{
    using S = typename DType<DT>::S;
    S *p = (S *)base + off;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (r.live >= (h + 1) * V) rot_store<DT, V>(p + r.at[h], v + h * V);
        else
#pragma unroll
            for (int i = 0; i < V; i++)
                if (h * V + i < r.live) p[r.at[h] + i] = DType<DT>::from_c(v[h * V + i]);
    }
}

// v turned by the angles of the unit's pairs, backwards with sign -1
template <int V, bool PAIRED>
__device__ __forceinline__ void rot_turn(const float2 *table, int u, float sign, float (&v)[2 * V])
{
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float2 cs = table[u * V + i];
        const int p = PAIRED ? 2 * i : i, q = PAIRED ? 2 * i + 1 : V + i;
        const float x = v[p], y = v[q], s = sign * cs.y;
        v[p] = x * cs.x - y * s;
        v[q] = x * s + y * cs.x;
    }
}

// the sum over the 2^log2 lanes that share a head
__device__ __forceinline__ float rot_sum(float v, int log2)
{
    for (int m = 1; m < 1 << log2; m <<= 1) v += __shfl_xor(v, m, PT_WAVE);
    return v;
}

// One block takes `group` tokens at a time and all heads of its side
// (blockIdx.y).  NU units a lane: two where a unit is one pair (heads of up
// to 256 elements then have 128 units).
template <int DT, int GDT, int V, bool PAIRED, bool BACK>
__global__ __launch_bounds__(kRotThreads) void k_rotary(RotArgs a)
{
    constexpr int NU = V == 1 ? 2 : 1;
    __shared__ float2 table[kRotTable];
    __shared__ float sums[BACK ? kRotThreads * NU * 2 * V : 1];
    const RotSide &s = a.side[blockIdx.y];
    const int log2 = a.lanes_log2, lane = threadIdx.x & ((1 << log2) - 1), slot = threadIdx.x >> log2;
    const int slots = kRotThreads >> log2, pairs = a.part / 2;
    RotUnit unit[NU];
    float w[NU][2 * V], dw[NU][2 * V];
#pragma unroll
    for (int k = 0; k < NU; k++) {
        unit[k] = rot_unit<V, PAIRED>(a, lane + (k << log2));
        if (s.scale) rot_read<DT, V>(s.scale, 0, unit[k], w[k]);
#pragma unroll
        for (int i = 0; i < 2 * V; i++) {
            if (!s.scale) w[k][i] = 1.0f;
            dw[k][i] = 0.0f;
        }
    }
    const float inv_n = 1.0f / (float)a.size;
    // (blocks times tokens of a group stay below 2^24 here, rows below 2^31)
    for (unsigned first = blockIdx.x * a.group; first < a.rows; first += gridDim.x * a.group) {
        const unsigned here = min((unsigned)a.group, a.rows - first);
        const unsigned items = here * (unsigned)s.heads;
        float x[NU][2 * V], g[NU][2 * V];
        long long to = 0;
        unsigned tok = 0;
        auto fetch = [&](unsigned item) {
            tok = item / (unsigned)s.heads;
            const unsigned head = item - tok * s.heads, row = first + tok, seq = row / a.tokens, t = row - seq * a.tokens;
            to = ((long long)row * s.heads + head) * a.size;
            const long long from = seq * s.st[0] + t * s.st[1] + head * s.st[2];
#pragma unroll
            for (int k = 0; k < NU; k++) {
                if (!BACK || s.scale) rot_read<DT, V>(s.x, from, unit[k], x[k]);
                if constexpr (BACK) rot_read<GDT, V>(s.g, to, unit[k], g[k]);
            }
        };
        unsigned item = slot;
        if (item < items) fetch(item);
        __syncthreads();  // the table's readers of the group before
        for (unsigned i = threadIdx.x; i < here * pairs; i += kRotThreads) {
            const unsigned tk = i / (unsigned)pairs, f = i - tk * pairs;
            const unsigned row = first + tk, seq = row / a.tokens, t = row - seq * a.tokens;
            const long long pos = a.positions ? (long long)a.positions[seq * a.pst[0] + t * a.pst[1]] : (long long)t;
            const double turns = (double)pos * a.turns[f];
            double sn, cs;
            sincospi(2.0 * (turns - rint(turns)), &sn, &cs);
            table[i] = make_float2((float)(cs * a.magnitude), (float)(sn * a.magnitude));
        }
        __syncthreads();
        // (whole groups of lanes enter and leave, so a head's sum has all its lanes)
        while (item < items) {
            const float2 *angles = table + tok * pairs;
            if constexpr (!BACK) {
                if (s.scale) {
                    float q = 0.0f;
#pragma unroll
                    for (int k = 0; k < NU; k++)
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) q = fmaf(x[k][i], x[k][i], q);
                    const float r = 1.0f / sqrtf(rot_sum(q, log2) * inv_n + a.eps);
#pragma unroll
                    for (int k = 0; k < NU; k++)
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) x[k][i] = x[k][i] * r * w[k][i];
                }
#pragma unroll
                for (int k = 0; k < NU; k++) {
                    if (unit[k].turned) rot_turn<V, PAIRED>(angles, lane + (k << log2), 1.0f, x[k]);
                    rot_write<DT, V>(s.y, to, unit[k], x[k]);
                }
            } else {
#pragma unroll
                for (int k = 0; k < NU; k++)
                    if (unit[k].turned) rot_turn<V, PAIRED>(angles, lane + (k << log2), -1.0f, g[k]);
                if (s.scale) {
                    float q = 0.0f, b = 0.0f;
#pragma unroll
                    for (int k = 0; k < NU; k++)
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) {
                            q = fmaf(x[k][i], x[k][i], q);
                            b = fmaf(g[k][i] * w[k][i], x[k][i], b);
                        }
                    const float r = 1.0f / sqrtf(rot_sum(q, log2) * inv_n + a.eps);
                    b = rot_sum(b, log2) * inv_n * r;
#pragma unroll
                    for (int k = 0; k < NU; k++)
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) {
                            const float u = x[k][i] * r;
                            dw[k][i] = fmaf(g[k][i], u, dw[k][i]);
                            g[k][i] = r * (g[k][i] * w[k][i] - u * b);
                        }
                }
#pragma unroll
                for (int k = 0; k < NU; k++)
                    if (s.y) rot_write<DT, V>(s.y, to, unit[k], g[k]);
            }
            item += slots;
            if (item < items) fetch(item);
        }
    }
    if constexpr (BACK) {
        if (!s.partial) return;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NU; k++)
#pragma unroll
            for (int i = 0; i < 2 * V; i++) sums[(k * 2 * V + i) * kRotThreads + threadIdx.x] = dw[k][i];
        __syncthreads();
        if (slot) return;
#pragma unroll
        for (int k = 0; k < NU; k++)
#pragma unroll
            for (int i = 0; i < 2 * V; i++) {
                float t = 0.0f;
                for (int o = 0; o < slots; o++) t += sums[(k * 2 * V + i) * kRotThreads + (o << log2) + lane];
                if (i < unit[k].live)
                    s.partial[(long long)blockIdx.x * a.size + unit[k].at[i / V] + i % V] = t;
            }
    }
}

// The scale's gradient from the blocks' partial rows, in a fixed order: four
// columns a block of 16 waves, a wave's lanes four columns and 16 rows.
template <int DT>
__global__ __launch_bounds__(256) void k_rotary_scale(RotArgs a, int parts, void *d0, void *d1)
{
    __shared__ float box[64][4];
    const int c = (int)blockIdx.x * 4 + (threadIdx.x & 3), r0 = threadIdx.x >> 2;
    void *out = blockIdx.y ? d1 : d0;
    const float *p = a.side[blockIdx.y].partial;
    if (!out) return;  // whole block
    float t = 0.0f;
    if (c < a.size)
        for (int r = r0; r < parts; r += 64) t += p[(long long)r * a.size + c];
    box[r0][threadIdx.x & 3] = t;
    __syncthreads();
    if (r0 || c >= a.size) return;
    for (int r = 1; r < 64; r++) t += box[r][threadIdx.x & 3];
    ((typename DType<DT>::S *)out)[c] = DType<DT>::from_c(t);
}

template <int DT, int GDT, int V>
static void launch_rotary(const RotArgs &a, bool interleaved, bool back, dim3 grid, hipStream_t s)
{
    if (back) {
        if (interleaved) k_rotary<DT, GDT, V, true, true><<<grid, kRotThreads, 0, s>>>(a);
        else k_rotary<DT, GDT, V, false, true><<<grid, kRotThreads, 0, s>>>(a);
        return;
    }
    if constexpr (DT == GDT) {
        if (interleaved) k_rotary<DT, DT, V, true, false><<<grid, kRotThreads, 0, s>>>(a);
        else k_rotary<DT, DT, V, false, false><<<grid, kRotThreads, 0, s>>>(a);
    }
}

template <int DT, int GDT>
static void launch_rotary_width(RotArgs a, bool interleaved, bool back, unsigned blocks, unsigned sides, hipStream_t s)
{
    constexpr int W = 16 / sizeof(typename DType<DT>::S);  // a pack of 16 bytes
    const int pairs = a.part / 2;
    const int v = pairs % W == 0 ? W : pairs % 2 == 0 ? 2 : 1;
    const int units = pairs / v + (a.size - a.part + 2 * v - 1) / (2 * v);
    a.lanes_log2 = 0;
    while (a.lanes_log2 < 6 && 1 << a.lanes_log2 < units) a.lanes_log2++;
    const dim3 grid(blocks, sides);
    if (v == W) launch_rotary<DT, GDT, W>(a, interleaved, back, grid, s);
    else if (v == 2) launch_rotary<DT, GDT, 2>(a, interleaved, back, grid, s);
    else launch_rotary<DT, GDT, 1>(a, interleaved, back, grid, s);
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
    // tokens of a group: enough pairs for a block's threads, as long as there
    // is a block for every CU and each of a few turns
    a.group = std::max(1, std::min({kRotThreads / (d->part / 2), 16, (int)std::min<long long>(rows / 2048, 16)}));
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
    const unsigned blocks = (unsigned)std::min<long long>(((long long)a.rows + a.group - 1) / a.group, 1 << 20);
    if (d->dtype == PT_FLOAT32) launch_rotary_width<PT_FLOAT32, PT_FLOAT32>(a, d->interleaved, false, blocks, sides, s);
    else if (d->dtype == PT_FLOAT16) launch_rotary_width<PT_FLOAT16, PT_FLOAT16>(a, d->interleaved, false, blocks, sides, s);
    else launch_rotary_width<PT_BFLOAT16, PT_BFLOAT16>(a, d->interleaved, false, blocks, sides, s);
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
    long long blocks = ((long long)a.rows + a.group - 1) / a.group;
    // a partial row a block: four blocks a CU walk the tokens
    blocks = std::min<long long>(blocks, partial ? 1024 : 1 << 20);
    void *scratch = nullptr;
    if (partial) {
        PT_TRY(scratch_alloc(&scratch, (size_t)blocks * 2 * a.size * sizeof(float), s));
        for (int i = 0; i < sides; i++)
            if (ds[i]) a.side[i].partial = (float *)scratch + (size_t)i * blocks * a.size;
    }
    const bool same = grad_dtype == d->dtype;
    if (d->dtype == PT_FLOAT32) launch_rotary_width<PT_FLOAT32, PT_FLOAT32>(a, d->interleaved, true, blocks, sides, s);
    else if (d->dtype == PT_FLOAT16) {
        if (same) launch_rotary_width<PT_FLOAT16, PT_FLOAT16>(a, d->interleaved, true, blocks, sides, s);
        else launch_rotary_width<PT_FLOAT16, PT_FLOAT32>(a, d->interleaved, true, blocks, sides, s);
    } else {
        if (same) launch_rotary_width<PT_BFLOAT16, PT_BFLOAT16>(a, d->interleaved, true, blocks, sides, s);
        else launch_rotary_width<PT_BFLOAT16, PT_FLOAT32>(a, d->interleaved, true, blocks, sides, s);
    }
    if (partial) {
        const dim3 grid((a.size + 3) / 4, sides);
        if (d->dtype == PT_FLOAT32) k_rotary_scale<PT_FLOAT32><<<grid, 256, 0, s>>>(a, (int)blocks, ds[0], ds[1]);
        else if (d->dtype == PT_FLOAT16) k_rotary_scale<PT_FLOAT16><<<grid, 256, 0, s>>>(a, (int)blocks, ds[0], ds[1]);
        else k_rotary_scale<PT_BFLOAT16><<<grid, 256, 0, s>>>(a, (int)blocks, ds[0], ds[1]);
    }
    const pt_status st = check_hip(hipGetLastError(), "rotary gradient");
    if (scratch) scratch_free(scratch, s);
    return st;
}

}  // extern "C"
