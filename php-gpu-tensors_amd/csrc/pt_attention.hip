// Attention over prompts and caches and its gradients: the C entries, their
// checks, the choice of kernel and split, and the small kernels around the
// ones of pt_attention.h.
#include "pt_attention.h"

#include <algorithm>
#include <math.h>
#include <type_traits>

namespace pt {

// A token of a sequence, and a head.
struct AttnToken {
    int b, i, h;
    long long row;  // in a packed tensor
};

// The token and head that this wave of a block of four takes.  Of a packed
// tensor with fewer rows than all sequences would have at the longest's
// length (`packed`), a token row, whose sequence the lanes look for; else one
// of that many.  Either fits 32 bits: split work is small.
__device__ __forceinline__ bool attn_wave_token(const AttnArgs &g, bool keys, bool packed, AttnToken &t)
{
    const int32_t *starts = keys ? g.k_starts : g.q_starts, *lengths = keys ? g.k_lengths : g.q_lengths;
    const int rows = keys ? g.k_rows : g.q_rows, most = keys ? g.nk : g.nq, heads = keys ? g.kv_heads : g.heads;
    const unsigned at = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), x = at / (unsigned)heads;
    t.h = (int)(at - x * heads);
    if (!packed) {
        t.b = (int)(x / (unsigned)most);
        t.i = (int)(x - (unsigned)t.b * most);
        if (t.b >= g.batch) return false;
        const AttnSeq s = attn_seq(starts, lengths, rows, most, t.b);
        t.row = s.row + t.i;
        return t.i < s.n;
    }
    if (x >= (unsigned)rows) return false;
    for (int c = 0; c < g.batch; c += 64) {
        const int b = c + (int)(threadIdx.x & 63);
        AttnSeq s = {0, 0};
        if (b < g.batch) s = attn_seq(starts, lengths, rows, most, b);
        const uint64_t in = __ballot(s.n && (long long)x >= s.row && (long long)x < s.row + s.n);
        if (!in) continue;
        const int lane = (int)__builtin_ctzll(in);
        t.b = c + lane;
        t.row = x;
        t.i = (int)x - __builtin_amdgcn_readlane((int)s.row, lane);
        return true;
    }
    return false;
}

// Is it, and blocks for it.
static bool attention_packed(const AttnArgs &g, bool keys)
{
    return keys ? g.k_starts && g.k_rows < (long long)g.batch * g.nk : g.q_starts && g.q_rows < (long long)g.batch * g.nq;
}
static dim3 attention_wave_tokens(const AttnArgs &g, bool keys, bool packed)
{
    const long long tokens = packed ? (keys ? g.k_rows : g.q_rows) : (long long)g.batch * (keys ? g.nk : g.nq);
    return dim3((unsigned)((tokens * (keys ? g.kv_heads : g.heads) + 3) / 4), keys ? 2 : 1);
}

// Joins the key ranges that workgroups of their own computed: with the
// common maximum m = max m_s, l = sum l_s 2^(m_s - m) and o = sum o_s
// 2^(m_s - m) / l.  One wave a row, at most 64 ranges; each part is read once.
template <int DT>
__global__ __launch_bounds__(256) void k_attention_join(AttnArgs g)
{
    const int lane = threadIdx.x & 63;
    AttnToken at;
    if (!attn_wave_token(g, false, g.part_packed, at)) return;
    const int b = at.b, qi = at.i, hq = at.h, hk = hq / g.group;
    // lane s holds range s
    const long long first = attn_part_row(g, b * g.kv_heads + hk, qi * g.group + hq % g.group, at.row, hq), step = g.part_step;
    float m = -INFINITY, l = 0.0f;
    if (lane < g.splits) {
        m = g.part_ml[(lane * step + first) * 2];
        l = g.part_ml[(lane * step + first) * 2 + 1];
    }
    // (attn_far_part: of a far row m is unscaled, and its parts are told apart by the exact difference)
    const float c = g.scale_log2;
    const bool far = l < 0.0f;
    l = fabsf(l);
    const float mc = far ? m * c : m, top = wave_all(mc, FMax{}), ref = top == -INFINITY ? 0.0f : top;
    float up = mc - ref;
    if (__any(far)) {
        const bool farthest = attn_far(top);  // then every part at the top is far
        const float most = wave_all(far && mc == top ? m : -INFINITY, FMax{});
        up = farthest ? (far ? (m - most) * c : -fmaf(most, c, -m)) : far ? fmaf(m, c, -ref) : up;
    }
    // a range in which the row sees nothing has written no sums
    const uint64_t some = __ballot(l != 0.0f);
    const float weight = __builtin_amdgcn_exp2f(up), sum = wave_all(l * weight, FAdd{});
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const long long to = b * g.o_bs + at.row * g.o_ts + hq * g.o_hs;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < g.splits; s++) {
        if (!(some >> s & 1)) continue;
        const float c = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), s));
        const float *from = g.part_o + (s * step + first) * g.size;
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (k * 64 + lane < g.size) x[k] = fmaf(from[k * 64 + lane], c, x[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
        if (k * 64 + lane < g.size) {
            store_c<DT>((typename AttnT<DT>::S *)g.out + to, (size_t)(k * 64 + lane), x[k] * inv);
            if constexpr (DT != PT_FLOAT32) {
                if (g.rest)
                    store_c<DT>((typename AttnT<DT>::S *)g.rest + to, (size_t)(k * 64 + lane), attn_rest<DT>(x[k] * inv));
            }
        }
    if (g.lse && lane == 0)
        g.lse[(g.q_starts ? at.row : (long long)b * g.heads * g.nq + qi) + (long long)hq * g.stat_rows] =
            sum == 0.0f ? -INFINITY : (ref + __builtin_amdgcn_logf(sum)) * 0.69314718055994531f;
}

// Adds the shares of a gradient that workgroups of their own computed, in
// their order: token rows of the queries (`keys` false: dq) or of the keys
// (dk, and dv), `heads` heads to a row.  One wave a row and head.
template <int DT>
__global__ __launch_bounds__(256) void k_attention_sum(AttnArgs g, bool keys, bool packed)
{
    const float *part = blockIdx.y ? g.part_ml : g.part_o;
    void *out = !keys ? g.dq : blockIdx.y ? g.dv : g.dk;
    const int lane = threadIdx.x & 63;
    AttnToken t;
    if (!attn_wave_token(g, keys, packed, t)) return;
    const long long row = (keys ? g.k_starts : g.q_starts) ? t.row : (long long)t.b * (keys ? g.nk : g.nq) + t.i;
    const long long to = (row * (keys ? g.kv_heads : g.heads) + t.h) * g.size;
    for (int d = lane; d < g.size; d += 64) {
        float x = 0.0f;
#pragma unroll 4
        for (int p = 0; p < g.splits; p++) x += part[p * g.part_step + to + d];
        store_c<DT>(out, (size_t)(to + d), x);
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
    // no sequence is longer than its tensor
    const int nq = d->q_starts ? std::min(d->queries, d->q_rows) : d->queries, nk = d->k_starts ? std::min(d->keys, d->k_rows) : d->keys;
    // (the last tile's rows are numbered past the last row)
    if (!fits_int((long long)nq * group + 255) || !fits_int(nk + 255ll) || !fits_int((long long)d->sequences * d->heads) ||
        !fits_int(((long long)nq * group / 32 + 1) * d->sequences * d->kv_heads) ||
        !fits_int(((long long)nk / 128 + 8) * d->sequences * 8 * d->kv_heads) ||
        !fits_int(((long long)nq * group / 128 + 8) * d->sequences * 8 * d->kv_heads))
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
    g.q_rows = d->q_rows;
    g.k_rows = d->k_rows;
    g.nq = nq;
    g.nk = nk;
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

// Key ranges of the forward pass.  A prompt's workgroups are split where they
// are fewer than the CUs; those of single tokens, which only read keys, until
// there are enough of them to even out caches of different lengths.  256 keys
// a range at least: a range costs a second kernel's read of its sums.
static int attention_splits(const AttnArgs &g, bool token, long long blocks)
{
    const long long most = std::min<long long>((g.nk + 255ll) / 256, 64);
    if (most <= 1) return 1;
    if (token) return (int)std::min<long long>(std::max<long long>(1, 2048 / blocks), most);
    // packed prompts have no more tiles than their rows fill
    if (g.q_starts) blocks = std::min(blocks, ((long long)g.q_rows * g.group / 128 + g.batch) * g.kv_heads);
    return blocks < 256 ? (int)std::min<long long>((512 + blocks - 1) / blocks, most) : 1;
}

// Shares of a gradient kernel with `blocks` workgroups of `steps` tiles each:
// enough to fill the CUs twice, four tiles to a share at least.
static int backward_splits(long long blocks, long long steps)
{
    if (blocks >= 256 || steps < 8) return 1;
    return (int)std::min<long long>(std::min<long long>((512 + blocks - 1) / blocks, steps / 4), 16);
}

// Sets the order of the workgroups for `tiles` tiles of 128 rows in the
// longest sequence and returns their number.  rows: of a packed tensor, which
// bound the tiles of all its sequences together; 0 for sequences of one length.
static long long attention_place(AttnArgs &g, long long tiles, long long rows, bool ragged)
{
    const long long nh = (long long)g.batch * g.kv_heads;
    const int share = 8 % g.kv_heads == 0 ? 8 / g.kv_heads : 0;
    g.tiles = (int)tiles;
    if (ragged) {
        g.place = kRagged;
        const long long items = std::min(tiles * g.batch, rows / 128 + g.batch);
        return share ? (items + share - 1) / share * 8 : items * g.kv_heads;
    }
    g.place = nh % 8 == 0 ? kGrouped : share ? kSpread : kPlain;
    return g.place == kSpread ? (tiles + share - 1) / share * 8 * g.batch : tiles * nh;
}

// Is it work for k_attention_token?
static bool attention_token(const AttnArgs &g, bool vec) { return (long long)g.nq * g.group <= 32 && vec; }

// Workgroups of the forward pass, of the queries' gradient and of the keys';
// each sets the order of the kernel that is launched next.
static long long forward_grid(AttnArgs &g, bool token, long long tiles)
{
    return token ? (long long)g.batch * g.kv_heads : attention_place(g, tiles, (long long)g.q_rows * g.group, g.q_starts);
}
static long long queries_grid(AttnArgs &g) { return forward_grid(g, false, ((long long)g.nq * g.group + 127) / 128); }
static long long keys_grid(AttnArgs &g) { return attention_place(g, ((long long)g.nk + 127) / 128, g.k_rows, g.k_starts); }

// A launch counts its threads, 256 a workgroup, in 32 bits.
static pt_status attention_launches(AttnArgs g, bool vec, bool backward)
{
    const long long most = 0xffffffffll / 256;
    const bool token = !backward && attention_token(g, vec);
    if (g.batch && g.nq && (token ? forward_grid(g, true, 1) : queries_grid(g)) > most)
        return fail(PT_ERR_INVALID, "attention has more tiles of queries than a launch holds");
    if (backward && g.batch && g.nk && keys_grid(g) > most)
        return fail(PT_ERR_INVALID, "attention has more tiles of keys than a launch holds");
    return PT_OK;
}

template <int DT> static pt_status attention_typed(AttnArgs &g, bool vec, hipStream_t s)
{
    const long long nh = (long long)g.batch * g.kv_heads, rows = (long long)g.nq * g.group;
    const bool token = attention_token(g, vec);
    const long long blocks = (rows + (token ? 31 : 127)) / (token ? 32 : 128) * nh;
    if (!blocks) return PT_OK;
    g.splits = attention_splits(g, token, blocks);
    void *scratch = nullptr;
    if (g.splits > 1) {
        // the longest of packed prompts may be much longer than most of them
        g.part_packed = attention_packed(g, false);
        g.part_step = g.part_packed ? (long long)g.q_rows * g.heads : nh * rows;
        const size_t parts = (size_t)g.splits * g.part_step;
        PT_TRY(scratch_alloc(&scratch, parts * (g.size + 2) * sizeof(float), s));
        g.part_ml = (float *)scratch;
        g.part_o = g.part_ml + parts * 2;
    }
    launch_attention<DT>(g, token, vec, (unsigned)forward_grid(g, token, blocks / nh), s);
    pt_status st = check_hip(hipGetLastError(), "attention");
    if (st == PT_OK && g.splits > 1) {
        k_attention_join<DT><<<attention_wave_tokens(g, false, g.part_packed), 256, 0, s>>>(g);
        st = check_hip(hipGetLastError(), "attention join");
    }
    if (scratch) scratch_free(scratch, s);
    return st;
}

template <int DT>
static pt_status attention_backward_typed(AttnArgs &g, bool vec, const void *w, bool w32, hipStream_t s)
{
    const long long nh = (long long)g.batch * g.kv_heads, rows = (long long)g.nq * g.group;
    const long long q_rows = g.q_starts ? g.q_rows : (long long)g.batch * g.nq, stats = q_rows * g.heads;
    const long long k_elems = (g.k_starts ? g.k_rows : (long long)g.batch * g.nk) * g.kv_heads * g.size;
    const bool round = w32 && DT != PT_FLOAT32;
    const long long kb = ((long long)g.nk + 127) / 128 * nh, qb = (rows + 127) / 128 * nh;
    const long long k_live = g.k_starts ? std::min(kb, ((long long)g.k_rows / 128 + g.batch) * g.kv_heads) : kb;
    const long long q_live = g.q_starts ? std::min(qb, ((long long)g.q_rows * g.group / 128 + g.batch) * g.kv_heads) : qb;
    const int tile = attention_backward_tile<DT>(g.size);
    const int k_splits = kb ? backward_splits(std::max(1ll, k_live), ((long long)g.nq + tile - 1) / tile * g.group) : 1;
    const int q_splits = qb ? backward_splits(std::max(1ll, q_live), ((long long)g.nk + tile - 1) / tile) : 1;
    // one region: lse2, delta, tops, the rounded upstream gradient, the shares (of
    // dq, and after them of dk and dv)
    auto whole = [](size_t n) { return (n + 255) & ~(size_t)255; };
    const size_t stat_bytes = whole((size_t)stats * 4), w_bytes = round ? whole((size_t)stats * g.size * 2) : 0;
    const size_t k_part = k_splits > 1 ? whole((size_t)k_splits * k_elems * 4) : 0;
    const size_t q_part = q_splits > 1 ? whole((size_t)q_splits * stats * g.size * 4) : 0;
    void *scratch = nullptr;
    PT_TRY(scratch_alloc(&scratch, 3 * stat_bytes + w_bytes + std::max(2 * k_part, q_part), s));
    char *base = (char *)scratch;
    g.lse2 = (float *)base;
    g.delta = (float *)(base + stat_bytes);
    g.tops = (float *)(base + 2 * stat_bytes);
    void *w16 = base + 3 * stat_bytes;
    float *part = (float *)(base + 3 * stat_bytes + w_bytes);
    pt_status st = PT_OK;
    if (round && stats) {
        // the products take 16-bit operands
        const int shape[4] = {g.q_starts ? 1 : g.batch, g.q_starts ? g.q_rows : g.nq, g.heads, g.size};
        const size_t strides[4] = {(size_t)g.o_ts * shape[1], (size_t)g.o_ts, (size_t)g.o_hs, 1};
        st = pt_cast(w, PT_FLOAT32, strides, 0, w16, DT, shape, 4, (pt_stream_t)s);
    }
    g.w = round ? w16 : w;
    vec = vec && !(((uintptr_t)g.w | (uintptr_t)g.out | (uintptr_t)g.rest) & 15);
    // the queries' pass leaves lse2 and d to the keys'
    if (st == PT_OK && qb) {
        g.splits = q_splits;
        g.part_step = stats * g.size;
        g.part_o = part;
        launch_attention_dq<DT>(g, vec, (unsigned)queries_grid(g), s);
        if (q_splits > 1) {
            const bool packed = attention_packed(g, false);
            k_attention_sum<DT><<<attention_wave_tokens(g, false, packed), 256, 0, s>>>(g, false, packed);
        }
        st = check_hip(hipGetLastError(), "attention gradient of queries");
    }
    if (st == PT_OK && kb) {
        g.splits = k_splits;
        g.part_step = k_elems;
        g.part_o = part;
        g.part_ml = (float *)((char *)part + k_part);
        launch_attention_dkv<DT>(g, vec, (unsigned)keys_grid(g), s);
        if (k_splits > 1) {
            const bool packed = attention_packed(g, true);
            k_attention_sum<DT><<<attention_wave_tokens(g, true, packed), 256, 0, s>>>(g, true, packed);
        }
        st = check_hip(hipGetLastError(), "attention gradient of keys and values");
    }
    scratch_free(scratch, s);
    return st;
}

}  // namespace pt

using namespace pt;

extern "C" {

pt_status pt_attention(const pt_attention_desc *desc, const void *q, const void *k, const void *v, void *out, float *lse,
                       void *rest, pt_stream_t stream)
{
    AttnArgs g;
    bool vec;
    PT_TRY(attention_args(desc, q, k, v, g, vec));
    if (!out && g.batch && g.nq && g.stat_rows) return fail(PT_ERR_INVALID, "attention output is missing");
    PT_TRY(attention_launches(g, vec, false));
    PT_TRY(ensure_init());
    g.out = out;
    g.lse = lse;
    g.rest = rest;
    hipStream_t s = stream_of(stream);
    switch (desc->dtype) {
    case PT_FLOAT32: return attention_typed<PT_FLOAT32>(g, vec, s);
    case PT_FLOAT16: return attention_typed<PT_FLOAT16>(g, vec, s);
    default: return attention_typed<PT_BFLOAT16>(g, vec, s);
    }
}

pt_status pt_attention_backward(const pt_attention_desc *desc, const void *q, const void *k, const void *v,
                                const void *out, const float *lse, const void *rest, const void *grad, int grad_dtype,
                                void *dq, void *dk, void *dv, pt_stream_t stream)
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
    PT_TRY(attention_launches(g, vec, true));
    PT_TRY(ensure_init());
    g.out = const_cast<void *>(out);
    g.rest = const_cast<void *>(rest);
    g.lse = const_cast<float *>(lse);
    g.dq = dq;
    g.dk = dk;
    g.dv = dv;
    hipStream_t s = stream_of(stream);
    const bool w32 = grad_dtype == PT_FLOAT32;
    switch (desc->dtype) {
    case PT_FLOAT32: return attention_backward_typed<PT_FLOAT32>(g, vec, grad, w32, s);
    case PT_FLOAT16: return attention_backward_typed<PT_FLOAT16>(g, vec, grad, w32, s);
    default: return attention_backward_typed<PT_BFLOAT16>(g, vec, grad, w32, s);
    }
}

}  // extern "C"
