// Attention over prompts and caches and its gradients: the C entries, their
// checks, the choice of kernel and split, and the small kernels around the
// ones of pt_attention.h.
#include "pt_attention.h"

#include <algorithm>
#include <math.h>

namespace pt {

// Joins the key ranges that workgroups of their own computed: with the
// common maximum m = max m_s, l = sum l_s 2^(m_s - m) and o = sum o_s
// 2^(m_s - m) / l.  One wave a row; it reads each part once.
template <int DT>
__global__ __launch_bounds__(256) void k_attention_join(AttnArgs g)
{
    const int lane = threadIdx.x & 63;
    const long long rows = (long long)g.nq * g.group, nh = (long long)g.batch * g.kv_heads;
    const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= nh * rows) return;
    const int bh = (int)(at / rows), row = (int)(at % rows), b = bh / g.kv_heads;
    const int qi = row / g.group, hq = bh % g.kv_heads * g.group + row % g.group;
    const AttnSeq sq = attn_seq(g.q_starts, g.q_lengths, g.q_rows, g.nq, b);
    if (qi >= sq.n) return;
    float m = -INFINITY, l = 0.0f;
    for (int s = 0; s < g.splits; s++) m = fmaxf(m, g.part_ml[((long long)s * nh * rows + at) * 2]);
    const float ref = m == -INFINITY ? 0.0f : m;
    for (int s = 0; s < g.splits; s++) {
        const float *ml = g.part_ml + ((long long)s * nh * rows + at) * 2;
        l += ml[1] * __builtin_amdgcn_exp2f(ml[0] - ref);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    typename AttnT<DT>::S *to = (typename AttnT<DT>::S *)g.out + b * g.o_bs + (sq.row + qi) * g.o_ts + hq * g.o_hs;
    for (int d = lane; d < g.size; d += 64) {
        float x = 0.0f;
        for (int s = 0; s < g.splits; s++) {
            const long long part = (long long)s * nh * rows + at;
            const float ls = g.part_ml[part * 2 + 1];
            // a range in which the row sees nothing has written no sums
            if (ls != 0.0f) x += g.part_o[part * g.size + d] * __builtin_amdgcn_exp2f(g.part_ml[part * 2] - ref);
        }
        store_c<DT>(to, (size_t)d, x * inv);
    }
    if (g.lse && lane == 0)
        g.lse[(g.q_starts ? sq.row : (long long)b * g.heads * g.nq) + (long long)hq * g.stat_rows + qi] =
            l == 0.0f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
}

// Per row and head, before the gradients: d = w . o in fp32, lse in base 2,
// and the upstream gradient in the element type where it came in float32
// (the products take 16-bit operands).  A row that sees no key gets lse +inf,
// so its exponentials are 0.  16 lanes a row; HBM-bound, one read of w and o.
template <int DT, bool W32>
__global__ __launch_bounds__(256) void k_attention_prepare(const void *w, const void *out, const float *lse,
                                                           uint16_t *w16, float *lse2, float *delta, long long rows,
                                                           int heads, int size, int queries, bool packed)
{
    using S = typename AttnT<DT>::S;
    const int lane = threadIdx.x & 15;
    const long long at = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (at >= rows * heads) return;
    float x = 0.0f;
    for (int d = lane; d < size; d += 16) {
        const long long e = at * size + d;
        float wv;
        if constexpr (W32) {
            wv = ((const float *)w)[e];
            if constexpr (DT != PT_FLOAT32) {
                const uint16_t h = DT == PT_BFLOAT16 ? float_to_bf16(wv) : float_to_f16(wv);
                w16[e] = h;
                wv = DType<DT>::to_c(h);
            }
        } else {
            wv = DType<DT>::to_c(((const S *)w)[e]);
        }
        x = fmaf(wv, DType<DT>::to_c(((const S *)out)[e]), x);
    }
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) x += __shfl_xor(x, m, 16);
    if (lane == 0) {
        const long long row = at / heads, h = at % heads;
        const long long stat = packed ? h * rows + row : (row / queries * heads + h) * queries + row % queries;
        const float l = lse[stat];
        delta[stat] = x;
        lse2[stat] = l == -INFINITY ? INFINITY : l * 1.4426950408889634f;
    }
}

// The largest work a pass may hold in 32-bit row and block numbers.
static bool fits_int(long long v) { return v >= 0 && v <= 0x7fffffff; }

static pt_status attention_args(const pt_attention_desc *d, const void *q, const void *k, const void *v, AttnArgs &g,
                                bool &vec)
{
    if (!d) return fail(PT_ERR_INVALID, "attention needs a description");
    if (d->dtype != PT_FLOAT32 && d->dtype != PT_FLOAT16 && d->dtype != PT_BFLOAT16)
        return fail(PT_ERR_INVALID, "attention requires float32, float16 or bfloat16 operands");
    if (d->sequences < 0 || d->queries < 0 || d->keys < 0 || d->heads < 1 || d->kv_heads < 1 || d->head_size < 1)
        return fail(PT_ERR_INVALID, "attention sizes must not be negative, heads and head size must be positive");
    if (d->heads % d->kv_heads)
        return fail(PT_ERR_INVALID, "attention needs a multiple of %d key heads for %d query heads", d->kv_heads, d->heads);
    if (d->head_size > 256) return fail(PT_ERR_UNSUPPORTED, "attention heads hold at most 256 elements, not %d", d->head_size);
    if (!(d->scale > 0.0) || !isfinite((float)d->scale) || (float)d->scale < 1e-30f || (float)d->scale > 1e30f)
        return fail(PT_ERR_INVALID, "attention scale must be finite and positive");
    if ((d->q_starts == nullptr) != (d->q_lengths == nullptr) || (d->k_starts == nullptr) != (d->k_lengths == nullptr))
        return fail(PT_ERR_INVALID, "attention sequences need starts and lengths together");
    if ((d->q_starts && d->q_rows < 0) || (d->k_starts && d->k_rows < 0))
        return fail(PT_ERR_INVALID, "attention row counts must not be negative");
    const int group = d->heads / d->kv_heads;
    if (!fits_int((long long)d->queries * group) || !fits_int((long long)d->sequences * d->heads) ||
        !fits_int(((long long)d->queries * group / 32 + 1) * d->sequences * d->kv_heads) ||
        !fits_int(((long long)d->keys / 128 + 1) * d->sequences * d->kv_heads))
        return fail(PT_ERR_INVALID, "attention has more rows than 32-bit numbers count");
    g = AttnArgs();
    g.q = q;
    g.k = k;
    g.v = v;
    g.q_bs = d->q_starts ? 0 : (long long)d->q_strides[0];
    g.q_ts = (long long)d->q_strides[1];
    g.q_hs = (long long)d->q_strides[2];
    g.k_bs = d->k_starts ? 0 : (long long)d->k_strides[0];
    g.k_ts = (long long)d->k_strides[1];
    g.k_hs = (long long)d->k_strides[2];
    g.v_bs = d->k_starts ? 0 : (long long)d->v_strides[0];
    g.v_ts = (long long)d->v_strides[1];
    g.v_hs = (long long)d->v_strides[2];
    g.q_starts = d->q_starts;
    g.q_lengths = d->q_lengths;
    g.k_starts = d->k_starts;
    g.k_lengths = d->k_lengths;
    g.batch = d->sequences;
    g.heads = d->heads;
    g.kv_heads = d->kv_heads;
    g.group = group;
    g.size = d->head_size;
    g.nq = d->queries;
    g.nk = d->keys;
    g.q_rows = d->q_rows;
    g.k_rows = d->k_rows;
    g.o_hs = g.size;
    g.o_ts = (long long)g.size * g.heads;
    g.o_bs = g.q_starts ? 0 : g.o_ts * g.nq;
    g.stat_rows = g.q_starts ? g.q_rows : g.nq;
    g.causal = d->causal != 0;
    g.scale = (float)d->scale;
    g.scale_log2 = (float)(d->scale * 1.4426950408889634);
    g.splits = 1;
    const size_t es = dtype_size(d->dtype);
    const size_t n_q = (size_t)g.stat_rows * (g.q_starts ? 1 : g.batch), n_k = (size_t)(g.k_starts ? g.k_rows : g.nk * (long long)g.batch);
    if (g.batch && g.nq && n_q && !q) return fail(PT_ERR_INVALID, "attention queries are missing");
    if (g.batch && g.nk && n_k && (!k || !v)) return fail(PT_ERR_INVALID, "attention keys or values are missing");
    auto whole = [&](long long s) { return (s * (long long)es) % 16 == 0; };
    vec = (g.size * es) % 16 == 0 && !(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) && whole(g.q_bs) && whole(g.q_ts) &&
          whole(g.q_hs) && whole(g.k_bs) && whole(g.k_ts) && whole(g.k_hs) && whole(g.v_bs) && whole(g.v_ts) && whole(g.v_hs) &&
          // a tile's rows lie within 2 GiB of its first
          g.q_ts < (1 << 22) && g.k_ts < (1 << 22) && g.v_ts < (1 << 22) && g.o_ts < (1 << 22);
    return PT_OK;
}

template <int DT> static pt_status attention_typed(AttnArgs &g, bool vec, hipStream_t s)
{
    const long long nh = (long long)g.batch * g.kv_heads, rows = (long long)g.nq * g.group;
    const bool narrow = rows <= 32 && attention_narrow_built<DT>(g.size);
    const long long blocks = (rows + (narrow ? 31 : 127)) / (narrow ? 32 : 128) * nh;
    if (!blocks) return PT_OK;
    // With fewer workgroups than CUs the keys are split between several, at
    // least 256 keys each, and joined by a second kernel.
    const long long most = (g.nk + 255) / 256;
    if (blocks < 256 && most > 1) g.splits = (int)std::min<long long>(std::min<long long>((512 + blocks - 1) / blocks, most), 64);
    void *scratch = nullptr;
    if (g.splits > 1) {
        const size_t parts = (size_t)g.splits * nh * rows;
        PT_TRY(scratch_alloc(&scratch, parts * (g.size + 2) * sizeof(float), s));
        g.part_ml = (float *)scratch;
        g.part_o = g.part_ml + parts * 2;
    }
    launch_attention<DT>(g, narrow, vec, (unsigned)blocks, s);
    pt_status st = check_hip(hipGetLastError(), "attention");
    if (st == PT_OK && g.splits > 1) {
        k_attention_join<DT><<<(unsigned)((nh * rows + 3) / 4), 256, 0, s>>>(g);
        st = check_hip(hipGetLastError(), "attention join");
    }
    if (scratch) scratch_free(scratch, s);
    return st;
}

template <int DT>
static pt_status attention_backward_typed(AttnArgs &g, bool vec, const void *w, bool w32, const float *lse, hipStream_t s)
{
    const long long nh = (long long)g.batch * g.kv_heads, rows = (long long)g.nq * g.group;
    const long long q_rows = g.q_starts ? g.q_rows : (long long)g.batch * g.nq, stats = q_rows * g.heads;
    const size_t stat_bytes = ((size_t)stats * 4 + 255) & ~(size_t)255;
    const bool round = w32 && DT != PT_FLOAT32;
    void *scratch = nullptr;
    PT_TRY(scratch_alloc(&scratch, 2 * stat_bytes + (round ? (size_t)stats * g.size * 2 : 0), s));
    float *lse2 = (float *)scratch, *delta = (float *)((char *)scratch + stat_bytes);
    uint16_t *w16 = round ? (uint16_t *)((char *)scratch + 2 * stat_bytes) : nullptr;
    pt_status st = PT_OK;
    if (stats) {
        const unsigned n = (unsigned)((stats + 15) / 16);
        const bool packed = g.q_starts != nullptr;
        if (w32)
            k_attention_prepare<DT, true><<<n, 256, 0, s>>>(w, g.out, lse, w16, lse2, delta, q_rows, g.heads, g.size, g.nq, packed);
        else
            k_attention_prepare<DT, false><<<n, 256, 0, s>>>(w, g.out, lse, w16, lse2, delta, q_rows, g.heads, g.size, g.nq, packed);
        st = check_hip(hipGetLastError(), "attention gradient preparation");
    }
    g.w = round ? (const void *)w16 : w;
    g.lse2 = lse2;
    g.delta = delta;
    vec = vec && !((uintptr_t)g.w & 15);
    const long long kb = ((long long)g.nk + 127) / 128 * nh, qb = (rows + 127) / 128 * nh;
    if (st == PT_OK && kb && g.dk) {
        launch_attention_dkv<DT>(g, vec, (unsigned)kb, s);
        st = check_hip(hipGetLastError(), "attention gradient of keys and values");
    }
    if (st == PT_OK && qb && g.dq) {
        launch_attention_dq<DT>(g, vec, (unsigned)qb, s);
        st = check_hip(hipGetLastError(), "attention gradient of queries");
    }
    scratch_free(scratch, s);
    return st;
}

}  // namespace pt

using namespace pt;

extern "C" {

pt_status pt_attention(const pt_attention_desc *desc, const void *q, const void *k, const void *v, void *out, float *lse,
                       pt_stream_t stream)
{
    AttnArgs g;
    bool vec;
    PT_TRY(attention_args(desc, q, k, v, g, vec));
    if (!out && g.batch && g.nq && g.stat_rows) return fail(PT_ERR_INVALID, "attention output is missing");
    PT_TRY(ensure_init());
    g.out = out;
    g.lse = lse;
    hipStream_t s = stream_of(stream);
    switch (desc->dtype) {
    case PT_FLOAT32: return attention_typed<PT_FLOAT32>(g, vec, s);
    case PT_FLOAT16: return attention_typed<PT_FLOAT16>(g, vec, s);
    default: return attention_typed<PT_BFLOAT16>(g, vec, s);
    }
}

pt_status pt_attention_backward(const pt_attention_desc *desc, const void *q, const void *k, const void *v,
                                const void *out, const float *lse, const void *grad, int grad_dtype, void *dq, void *dk,
                                void *dv, pt_stream_t stream)
{
    AttnArgs g;
    bool vec;
    PT_TRY(attention_args(desc, q, k, v, g, vec));
    if (grad_dtype != desc->dtype && grad_dtype != PT_FLOAT32)
        return fail(PT_ERR_INVALID, "attention's upstream gradient must be float32 or of the operands' dtype");
    const bool any_q = g.batch && g.nq && g.stat_rows, any_k = g.batch && g.nk && (!g.k_starts || g.k_rows);
    if (any_q && (!out || !lse || !grad || !dq)) return fail(PT_ERR_INVALID, "attention backward misses an operand");
    if ((dk == nullptr) != (dv == nullptr) || (any_k && !dk))
        return fail(PT_ERR_INVALID, "attention backward misses the gradient of keys or values");
    PT_TRY(ensure_init());
    g.out = const_cast<void *>(out);
    g.dq = dq;
    g.dk = dk;
    g.dv = dv;
    hipStream_t s = stream_of(stream);
    const bool w32 = grad_dtype == PT_FLOAT32;
    switch (desc->dtype) {
    case PT_FLOAT32: return attention_backward_typed<PT_FLOAT32>(g, vec, grad, w32, lse, s);
    case PT_FLOAT16: return attention_backward_typed<PT_FLOAT16>(g, vec, grad, w32, lse, s);
    default: return attention_backward_typed<PT_BFLOAT16>(g, vec, grad, w32, lse, s);
    }
}

}  // extern "C"
