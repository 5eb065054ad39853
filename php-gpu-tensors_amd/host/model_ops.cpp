// Dispatch of the operators of language models: attention, the gradients of
// layerNorm, and the log probabilities of tokens.  Each checks its operands,
// allocates its results and launches through the C-ABI; inside a Fusion
// scope it records one native step, whose further results are buffers that
// the step writes (NAT_BUFFER / NAT_RESULT).
#include "runtime.hpp"

#include <limits.h>
#include <math.h>
#include <string.h>

#include <algorithm>

namespace phpt {

bool low_or_f32(int dt) { return dt == PT_FLOAT32 || dt == PT_FLOAT16 || dt == PT_BFLOAT16; }

bool same_shape(const Tensor &a, const Tensor &b)
{
    return a.ndims == b.ndims && std::equal(a.shape, a.shape + a.ndims, b.shape);
}

static bool clear(const TensorP &t)
{
    pt_scalar_t zero;
    memset(&zero, 0, sizeof(zero));
    zero.dtype = t->dtype;
    return check_status(pt_fill(t->data(), t->dtype, t->numel(), &zero, nullptr), "fill");
}

TensorP record_buffer(const int *shape, int nd, int dtype)
{
    NativeSpec sp;
    sp.kind = NAT_BUFFER;
    return fusion_record_native(sp, {}, shape, nd, dtype);
}

TensorP record_result(const TensorP &buffer, const TensorP &main)
{
    NativeSpec sp;
    sp.kind = NAT_RESULT;
    return fusion_record_native(sp, {buffer, main}, buffer->shape, buffer->ndims, buffer->dtype);
}

// -------------------------------------------------------------- sequences
const int32_t *Sequences::device_starts() const { return (const int32_t *)device->data(); }
const int32_t *Sequences::device_lengths() const { return (const int32_t *)device->data() + count(); }

SequencesP make_sequences(const int *lengths, const int *starts, int count)
{
    if (count < 1) {
        set_invalid("Sequences need at least one length");
        return nullptr;
    }
    auto s = std::make_shared<Sequences>();
    long long at = 0;
    for (int i = 0; i < count; i++) {
        const long long from = starts ? starts[i] : at;
        if (lengths[i] < 0 || from < 0) {
            set_invalid("Sequence lengths and starts must not be negative");
            return nullptr;
        }
        if (from + lengths[i] > INT_MAX) {
            set_invalid("Sequences hold at most %d rows", INT_MAX);
            return nullptr;
        }
        s->starts.push_back((int)from);
        s->lengths.push_back(lengths[i]);
        at = from + lengths[i];
        s->most = std::max(s->most, lengths[i]);
        if (lengths[i]) s->end = std::max(s->end, at);
        s->total += lengths[i];
    }
    std::vector<int> order;
    for (int i = 0; i < count; i++)
        if (lengths[i]) order.push_back(i);
    std::sort(order.begin(), order.end(), [&](int a, int b) { return s->starts[a] < s->starts[b]; });
    for (size_t i = 1; i < order.size(); i++)
        if (s->starts[order[i]] < s->starts[order[i - 1]] + s->lengths[order[i - 1]]) s->overlap = true;
    std::vector<int> both(s->starts);
    both.insert(both.end(), s->lengths.begin(), s->lengths.end());
    const int shape[2] = {2, count};
    s->device = from_host(both.data(), shape, 2, PT_INT32);
    return s->device ? s : nullptr;
}

// -------------------------------------------------------------- attention
// Checks that need no device, and the description without addresses.
static bool attention_desc(const TensorP &q, const TensorP &k, const TensorP &v, bool causal, double scale,
                           const SequencesP &qs, const SequencesP &ks, pt_attention_desc &d)
{
    if (!q || !k || !v) {
        set_invalid("Missing tensor operand");
        return false;
    }
    if (!low_or_f32(q->dtype) || k->dtype != q->dtype || v->dtype != q->dtype) {
        set_invalid("attention requires matching float32, float16 or bfloat16 operands");
        return false;
    }
    const int nd = q->ndims;
    if ((nd != 3 && nd != 4) || k->ndims != nd || !same_shape(*k, *v)) {
        set_invalid("attention requires queries, keys and values [tokens, heads, size] or [sequences, tokens, heads, size], "
                    "keys and values of one shape");
        return false;
    }
    const int heads = q->shape[nd - 2], kv = k->shape[nd - 2], size = q->shape[nd - 1];
    if (size != k->shape[nd - 1] || size < 1 || size > 256) {
        set_invalid("attention heads must have one size of 1 to 256 elements");
        return false;
    }
    if (heads < 1 || kv < 1 || heads % kv) {
        set_invalid("attention needs a number of query heads that is a multiple of the key heads");
        return false;
    }
    if (nd == 4 && q->shape[0] != k->shape[0]) {
        set_invalid("attention needs as many sequences of keys as of queries");
        return false;
    }
    if (scale == 0.0) scale = 1.0 / sqrt((double)size);
    if (!isfinite(scale) || scale < 1e-30 || scale > 1e30) {
        set_invalid("attention scale must be finite and positive");
        return false;
    }
    if (qs || ks) {
        if (nd != 3) {
            set_invalid("attention with sequences takes operands [tokens, heads, size]");
            return false;
        }
        if (!qs || !ks || qs->count() != ks->count()) {
            set_invalid("attention needs as many sequences of keys as of queries");
            return false;
        }
        if (qs->end > q->shape[0] || ks->end > k->shape[0]) {
            set_invalid("attention sequences reach past the tensor's tokens");
            return false;
        }
        if (qs->overlap) {
            set_invalid("attention query sequences must not overlap");
            return false;
        }
    }
    memset(&d, 0, sizeof(d));
    d.dtype = q->dtype;
    d.heads = heads;
    d.kv_heads = kv;
    d.head_size = size;
    d.causal = causal;
    d.scale = scale;
    d.sequences = qs ? qs->count() : nd == 4 ? q->shape[0] : 1;
    d.queries = qs ? qs->most : q->shape[nd - 3];
    d.keys = ks ? ks->most : k->shape[nd - 3];
    if (qs) {
        d.q_starts = qs->device_starts();
        d.q_lengths = qs->device_lengths();
        d.k_starts = ks->device_starts();
        d.k_lengths = ks->device_lengths();
        d.q_rows = q->shape[0];
        d.k_rows = k->shape[0];
    }
    return true;
}

// The operand itself where a head's elements lie side by side, else packed.
TensorP head_operand(const TensorP &t, size_t strides[3])
{
    TensorP u = t;
    const int nd = t->ndims;
    if (t->shape[nd - 1] > 1 && t->strides[nd - 1] != 1) {
        u = materialize(t);
        if (!u) return nullptr;
    }
    strides[0] = nd == 4 ? u->strides[0] : 0;
    strides[1] = u->strides[nd - 3];
    strides[2] = u->strides[nd - 2];
    return u;
}

static int lse_shape(const Tensor &q, int *shape)
{
    int n = 0;
    if (q.ndims == 4) shape[n++] = q.shape[0];
    shape[n++] = q.shape[q.ndims - 2];
    shape[n++] = q.shape[q.ndims - 3];
    return n;
}

static bool attention_run(const TensorP &q, const TensorP &k, const TensorP &v, bool causal, double scale,
                          const SequencesP &qs, const SequencesP &ks, const TensorP &out, const TensorP &lse,
                          const TensorP &rest)
{
    pt_attention_desc d;
    if (!attention_desc(q, k, v, causal, scale, qs, ks, d)) return false;
    TensorP a = head_operand(q, d.q_strides), b = head_operand(k, d.k_strides), c = head_operand(v, d.v_strides);
    if (!a || !b || !c) return false;
    // rows of no sequence are zeros
    if (qs && !qs->cover(q->shape[0]) && !clear(out)) return false;
    return check_status(pt_attention(&d, a->data(), b->data(), c->data(), out->data(), lse ? (float *)lse->data() : nullptr,
                                     rest ? rest->data() : nullptr, nullptr),
                        "Attention kernel failed");
}

bool cuda_array_attention(const TensorP &q, const TensorP &k, const TensorP &v, bool causal, double scale,
                          const SequencesP &qs, const SequencesP &ks, bool keep, TensorP out[3])
{
    pt_attention_desc d;
    if (!attention_desc(q, k, v, causal, scale, qs, ks, d)) return false;
    int ls[kMaxDims];
    const int ln = lse_shape(*q, ls);
    out[1] = out[2] = nullptr;
    const bool rest = keep && q->dtype != PT_FLOAT32;
    if (fusion_active()) {
        NativeSpec sp;
        sp.kind = NAT_ATTENTION;
        sp.causal = causal;
        sp.eps = scale;
        sp.q_seq = qs;
        sp.k_seq = ks;
        std::vector<TensorP> ins = {q, k, v};
        for (int i = 0; i < keep + rest; i++) {
            ins.push_back(i ? record_buffer(q->shape, q->ndims, q->dtype) : record_buffer(ls, ln, PT_FLOAT32));
            if (!ins.back()) return false;
        }
        out[0] = fusion_record_native(sp, ins, q->shape, q->ndims, q->dtype);
        for (int i = 0; out[0] && i < keep + rest; i++)
            if (!(out[1 + i] = record_result(ins[3 + i], out[0]))) return false;
        return out[0] != nullptr;
    }
    if (!guard(q) || !guard(k) || !guard(v)) return false;
    out[0] = output_tensor(q->shape, q->ndims, q->dtype);
    if (out[0] && keep) out[1] = make_empty(ls, ln, PT_FLOAT32);
    if (out[0] && rest) out[2] = make_empty(q->shape, q->ndims, q->dtype);
    if (!out[0] || (keep && !out[1]) || (rest && !out[2])) return false;
    return attention_run(q, k, v, causal, scale, qs, ks, out[0], out[1], out[2]);
}

// in: q, k, v, the output, lse, the upstream gradient, rest (or null)
static bool attention_backward_run(const TensorP *in, bool causal, double scale, const SequencesP &qs, const SequencesP &ks,
                                   const TensorP *out)
{
    const TensorP &q = in[0], &k = in[1], &v = in[2];
    pt_attention_desc d;
    if (!attention_desc(q, k, v, causal, scale, qs, ks, d)) return false;
    TensorP a = head_operand(q, d.q_strides), b = head_operand(k, d.k_strides), c = head_operand(v, d.v_strides);
    TensorP o = materialize(in[3]), lse = materialize(in[4]), g = materialize(in[5]);
    TensorP rest = in[6] ? materialize(in[6]) : nullptr;
    if (!a || !b || !c || !o || !lse || !g || (in[6] && !rest)) return false;
    if (qs && !qs->cover(q->shape[0]) && !clear(out[0])) return false;
    if (ks && !ks->cover(k->shape[0]) && (!clear(out[1]) || !clear(out[2]))) return false;
    return check_status(pt_attention_backward(&d, a->data(), b->data(), c->data(), o->data(), (const float *)lse->data(),
                                              rest ? rest->data() : nullptr, g->data(), g->dtype, out[0]->data(), out[1]->data(), out[2]->data(), nullptr),
                        "Attention gradient kernel failed");
}

bool cuda_array_attention_backward(const TensorP &q, const TensorP &k, const TensorP &v, const TensorP &o,
                                   const TensorP &lse, const TensorP &rest, const TensorP &grad, bool causal,
                                   double scale, const SequencesP &qs, const SequencesP &ks, TensorP out[3])
{
    pt_attention_desc d;
    if (!attention_desc(q, k, v, causal, scale, qs, ks, d)) return false;
    if (ks && ks->overlap) {
        set_invalid("attention gradients need key sequences that do not overlap");
        return false;
    }
    int ls[kMaxDims];
    const int ln = lse_shape(*q, ls);
    if (!o || !lse || !grad || !same_shape(*o, *q) || o->dtype != q->dtype || lse->dtype != PT_FLOAT32 || lse->ndims != ln ||
        !std::equal(ls, ls + ln, lse->shape) ||
        (rest && (q->dtype == PT_FLOAT32 || !same_shape(*rest, *q) || rest->dtype != q->dtype))) {
        set_invalid("attention gradients need the forward pass's results");
        return false;
    }
    if (!same_shape(*grad, *q) || (grad->dtype != q->dtype && grad->dtype != PT_FLOAT32)) {
        set_invalid("attention's upstream gradient must have the output's shape, in float32 or its dtype");
        return false;
    }
    if (fusion_active()) {
        NativeSpec sp;
        sp.kind = NAT_ATTENTION_BACKWARD;
        sp.causal = causal;
        sp.eps = scale;
        sp.q_seq = qs;
        sp.k_seq = ks;
        TensorP dk = record_buffer(k->shape, k->ndims, k->dtype), dv = dk ? record_buffer(v->shape, v->ndims, v->dtype) : nullptr;
        if (!dv) return false;
        std::vector<TensorP> ins = {q, k, v, o, lse, grad, dk, dv};
        if (rest) ins.push_back(rest);
        out[0] = fusion_record_native(sp, ins, q->shape, q->ndims, q->dtype);
        if (!out[0]) return false;
        out[1] = record_result(dk, out[0]);
        out[2] = record_result(dv, out[0]);
        return out[1] && out[2];
    }
    const TensorP in[7] = {q, k, v, o, lse, grad, rest};
    for (const TensorP &t : in)
        if (t && !guard(t)) return false;
    out[0] = output_tensor(q->shape, q->ndims, q->dtype);
    out[1] = make_empty(k->shape, k->ndims, k->dtype);
    out[2] = make_empty(v->shape, v->ndims, v->dtype);
    if (!out[0] || !out[1] || !out[2]) return false;
    return attention_backward_run(in, causal, scale, qs, ks, out);
}

// -------------------------------------------------- gradients of layerNorm
// `out` holds the results' tensors (null: not wanted).  The normalized axes
// go last in ascending order, as in the forward pass; its checks have run.
static bool layernorm_backward_run(const TensorP &a, const TensorP &grad, const int *axes_in, int naxes, double eps,
                                   const TensorP &scale, const TensorP &bias, TensorP *out)
{
    int axes[kMaxDims], sorted[kMaxDims], perm[kMaxDims], inv[kMaxDims], k = 0;
    bool seen[kMaxDims] = {false};
    for (int i = 0; i < naxes; i++) {
        axes[i] = sorted[i] = axes_in[i] < 0 ? axes_in[i] + a->ndims : axes_in[i];
        seen[axes[i]] = true;
    }
    std::sort(sorted, sorted + naxes);
    for (int d = 0; d < a->ndims; d++)
        if (!seen[d]) perm[k++] = d;
    for (int i = 0; i < naxes; i++) perm[k++] = sorted[i];
    bool identity = true;
    for (int d = 0; d < a->ndims; d++) {
        identity = identity && perm[d] == d;
        inv[perm[d]] = d;
    }
    int pperm[kMaxDims], pinv[kMaxDims];
    bool pidentity = true;
    for (int i = 0; i < naxes; i++)
        for (int j = 0; j < naxes; j++)
            if (axes[j] == sorted[i]) {
                pperm[i] = j;
                pinv[j] = i;
                pidentity = pidentity && i == j;
            }
    int cdt = a->dtype == PT_FLOAT64 ? PT_FLOAT64 : PT_FLOAT32;
    if ((scale && scale->dtype == PT_FLOAT64) || (bias && bias->dtype == PT_FLOAT64)) cdt = PT_FLOAT64;
    const bool half = a->dtype == PT_FLOAT16 || a->dtype == PT_BFLOAT16;
    TensorP x = a;
    if (half && cdt == PT_FLOAT64) x = tensor_cast(a, PT_FLOAT64);
    auto rows_of = [&](TensorP t) -> TensorP {
        if (t && !identity) t = transpose(t, perm, t->ndims);
        return t ? materialize(t) : nullptr;
    };
    x = rows_of(x);
    TensorP g = rows_of(tensor_cast(grad, cdt));
    if (!x || !g) return false;
    auto own = [&](const TensorP &p) { return !p || p->dtype == x->dtype; };
    const int pdt = cdt == PT_FLOAT32 && half && (scale || bias) && own(scale) && own(bias) ? x->dtype : cdt;
    TensorP gamma;
    if (scale) {
        gamma = tensor_cast(scale, pdt);
        if (gamma && !pidentity) gamma = transpose(gamma, pperm, naxes);
        gamma = gamma ? materialize(gamma) : nullptr;
        if (!gamma) return false;
    }
    size_t n = 1;
    int pshape[kMaxDims];
    for (int i = 0; i < naxes; i++) {
        pshape[i] = a->shape[sorted[i]];
        n *= (size_t)pshape[i];
    }
    // straight into the results where their layout and dtype are the kernel's
    TensorP raw[3];
    if (out[0]) raw[0] = identity && x->dtype == a->dtype ? out[0] : make_empty(x->shape, x->ndims, x->dtype);
    for (int i = 1; i < 3; i++)
        if (out[i]) raw[i] = pidentity && out[i]->dtype == pdt ? out[i] : make_empty(pshape, naxes, pdt);
    for (int i = 0; i < 3; i++)
        if (out[i] && !raw[i]) return false;
    const size_t rows = n ? a->numel() / n : 0;
    if (!check_status(pt_layernorm_backward(x->data(), g->data(), x->dtype, cdt, rows, n, eps,
                                            gamma ? gamma->data() : nullptr, pdt, raw[0] ? raw[0]->data() : nullptr,
                                            raw[1] ? raw[1]->data() : nullptr, raw[2] ? raw[2]->data() : nullptr, nullptr),
                      "LayerNorm gradient kernel failed"))
        return false;
    for (int i = 0; i < 3; i++) {
        if (!out[i] || raw[i] == out[i] || !out[i]->numel()) continue;
        TensorP t = raw[i];
        if (i == 0 ? !identity : !pidentity) t = transpose(t, i == 0 ? inv : pinv, t->ndims);
        if (!t || !check_status(pt_cast(t->storage->ptr, t->dtype, t->strides, t->offset, out[i]->data(), out[i]->dtype,
                                        t->shape, t->ndims, nullptr),
                                "LayerNorm gradient copy failed"))
            return false;
    }
    return true;
}

bool cuda_array_layernorm_backward(const TensorP &a, const TensorP &grad, const int *axes, int naxes, double eps,
                                   const TensorP &scale, const TensorP &bias, TensorP out[3])
{
    if (a && !is_floating(a->dtype)) {
        // whole numbers are normalized as float64, and have no gradient of their own
        TensorP f = tensor_cast(a, PT_FLOAT64);
        if (!f || !cuda_array_layernorm_backward(f, grad, axes, naxes, eps, scale, bias, out)) return false;
        out[0] = nullptr;
        return true;
    }
    if (!a || !grad || !same_shape(*a, *grad) || !is_floating(grad->dtype)) {
        set_invalid("LayerNorm gradients need a floating input and an upstream gradient of its shape");
        return false;
    }
    int checked[kMaxDims];
    if (!layernorm_axes(a, axes, naxes, eps, scale, bias, checked)) return false;
    if (fusion_active()) {
        NativeSpec sp;
        sp.kind = NAT_LAYERNORM_BACKWARD;
        sp.eps = eps;
        sp.naxes = naxes;
        for (int i = 0; i < naxes; i++) sp.axes[i] = axes[i];
        sp.has_scale = scale != nullptr;
        sp.has_bias = bias != nullptr;
        std::vector<TensorP> ins = {a, grad};
        TensorP box[3];
        const TensorP *params[3] = {nullptr, &scale, &bias};
        for (int i = 1; i < 3; i++)
            if (*params[i]) ins.push_back(*params[i]);
        for (int i = 1; i < 3; i++)
            if (const TensorP &p = *params[i]) {
                box[i] = record_buffer(p->shape, p->ndims, p->dtype);
                if (!box[i]) return false;
                ins.push_back(box[i]);
            }
        out[0] = fusion_record_native(sp, ins, a->shape, a->ndims, a->dtype);
        if (!out[0]) return false;
        for (int i = 1; i < 3; i++)
            if (box[i] && !(out[i] = record_result(box[i], out[0]))) return false;
        return true;
    }
    if (!guard(a) || !guard(grad) || (scale && !guard(scale)) || (bias && !guard(bias))) return false;
    out[0] = output_tensor(a->shape, a->ndims, a->dtype);
    out[1] = scale ? make_empty(scale->shape, scale->ndims, scale->dtype) : nullptr;
    out[2] = bias ? make_empty(bias->shape, bias->ndims, bias->dtype) : nullptr;
    if (!out[0] || (scale && !out[1]) || (bias && !out[2])) return false;
    return layernorm_backward_run(a, grad, axes, naxes, eps, scale, bias, out);
}

// -------------------------------------------------------- log probabilities
static bool logprobs_shapes(const TensorP &a, const TensorP &tokens, int top, int *rows, int *nr, int *tops)
{
    if (!a || !tokens) {
        set_invalid("Missing tensor operand");
        return false;
    }
    if (!low_or_f32(a->dtype) || a->ndims < 1) {
        set_invalid("logProbs requires float32, float16 or bfloat16 scores with classes along the last axis");
        return false;
    }
    *nr = std::max(1, a->ndims - 1);
    rows[0] = 1;
    for (int d = 0; d + 1 < a->ndims; d++) rows[d] = a->shape[d];
    if (tokens->dtype != PT_INT32 || tokens->ndims != *nr || !std::equal(rows, rows + *nr, tokens->shape)) {
        set_invalid("logProbs tokens must be int32, one for each row of scores");
        return false;
    }
    const int classes = a->shape[a->ndims - 1];
    if (classes < 1) {
        set_invalid("logProbs needs at least one class");
        return false;
    }
    if (top < 0 || top > 64 || top > classes) {
        set_invalid("logProbs lists 0 to 64 alternatives, and no more than the classes");
        return false;
    }
    // at most 9 axes of rows: one more fits
    for (int d = 0; d < *nr; d++) tops[d] = rows[d];
    tops[*nr] = top;
    return true;
}

// Scores whose rows lie one pitch apart, as they are; others packed.
static TensorP score_rows(const TensorP &a, size_t *rows, size_t *pitch)
{
    const int nd = a->ndims;
    size_t n = 1;
    for (int d = 0; d + 1 < nd; d++) n *= (size_t)a->shape[d];
    *rows = n;
    const size_t classes = (size_t)a->shape[nd - 1];
    *pitch = classes;
    bool plain = a->shape[nd - 1] == 1 || a->strides[nd - 1] == 1;
    size_t step = 0;  // of the innermost row axis that has several rows
    size_t inner = 1;
    for (int d = nd - 2; d >= 0 && plain; d--) {
        if (a->shape[d] == 1) continue;
        if (!step) {
            step = a->strides[d];
            plain = step >= classes;
            inner = (size_t)a->shape[d];
            continue;
        }
        plain = a->strides[d] == step * inner;
        inner *= (size_t)a->shape[d];
    }
    if (!plain) return materialize(a);
    if (step) *pitch = step;
    return a;
}

static bool logprobs_run(const TensorP &a, const TensorP &tokens, int top, const TensorP *out)
{
    size_t rows, pitch;
    TensorP x = score_rows(a, &rows, &pitch), t = materialize(tokens);
    if (!x || !t) return false;
    auto f = [&](int i) { return out[i] ? (float *)out[i]->data() : nullptr; };
    return check_status(pt_logprobs(x->data(), x->dtype, rows, (size_t)a->shape[a->ndims - 1], pitch,
                                    (const int32_t *)t->data(), top, f(0), f(1), f(2), f(3), (int32_t *)f(4), nullptr),
                        "Log probability kernel failed");
}

bool cuda_array_logprobs(const TensorP &a, const TensorP &tokens, int top, TensorP out[5])
{
    int rows[kMaxDims], tops[kMaxDims], nr;
    if (!logprobs_shapes(a, tokens, top, rows, &nr, tops)) return false;
    int pairs[kMaxDims];
    std::copy(tops, tops + nr, pairs);
    pairs[nr] = 2;
    if (fusion_active()) {
        NativeSpec sp;
        sp.kind = NAT_LOGPROBS;
        sp.top = top;
        std::vector<TensorP> ins = {a, tokens};
        TensorP box[5];
        for (int i = 1; i < (top ? 5 : 3); i++) {
            box[i] = i == 1 ? record_buffer(rows, nr, PT_FLOAT32)
                            : record_buffer(i == 2 ? pairs : tops, nr + 1, i == 4 ? PT_INT32 : PT_FLOAT32);
            if (!box[i]) return false;
            ins.push_back(box[i]);
        }
        out[0] = fusion_record_native(sp, ins, rows, nr, PT_FLOAT32);
        if (!out[0]) return false;
        for (int i = 1; i < 5; i++)
            if (box[i] && !(out[i] = record_result(box[i], out[0]))) return false;
        return true;
    }
    if (!guard(a) || !guard(tokens)) return false;
    out[0] = output_tensor(rows, nr, PT_FLOAT32);
    out[1] = make_empty(rows, nr, PT_FLOAT32);
    out[2] = make_empty(pairs, nr + 1, PT_FLOAT32);
    for (int i = 3; i < 5; i++) out[i] = top ? make_empty(tops, nr + 1, i == 3 ? PT_FLOAT32 : PT_INT32) : nullptr;
    for (int i = 0; i < (top ? 5 : 3); i++)
        if (!out[i]) return false;
    return logprobs_run(a, tokens, top, out);
}

// in: scores, tokens, stats, entropy, then as `given` says (bits): 1 the
// indices of the alternatives, 2, 4 and 8 the upstream gradients of the log
// probability, the entropy and the alternatives
static bool logprobs_backward_run(const std::vector<TensorP> &in, int given, const TensorP &out)
{
    size_t rows, pitch;
    TensorP x = score_rows(in[0], &rows, &pitch);
    if (!x) return false;
    TensorP part[7];  // tokens, stats, entropy, index, three gradients
    size_t at = 1;
    for (int i = 0; i < 7; i++) {
        if (i >= 3 && !(given >> (i - 3) & 1)) continue;
        part[i] = materialize(in[at++]);
        if (!part[i]) return false;
    }
    auto f = [&](int i) { return part[i] ? (const float *)part[i]->data() : nullptr; };
    const int top = part[3] ? part[3]->shape[part[3]->ndims - 1] : 0;
    return check_status(pt_logprobs_backward(x->data(), x->dtype, rows, (size_t)in[0]->shape[in[0]->ndims - 1], pitch,
                                             (const int32_t *)f(0), top, (const int32_t *)f(3), f(1), f(2), f(4), f(5), f(6),
                                             out->data(), nullptr),
                        "Log probability gradient kernel failed");
}

TensorP cuda_array_logprobs_backward(const TensorP &a, const TensorP &tokens, const TensorP &stats, const TensorP &entropy,
                                     const TensorP &top_index, const TensorP &g_logprob, const TensorP &g_entropy,
                                     const TensorP &g_top)
{
    int rows[kMaxDims], tops[kMaxDims], nr;
    const int top = top_index && top_index->ndims ? top_index->shape[top_index->ndims - 1] : 0;
    if (!logprobs_shapes(a, tokens, top, rows, &nr, tops)) return nullptr;
    auto row_value = [&](const TensorP &t) {
        return !t || (t->dtype == PT_FLOAT32 && t->ndims == nr && std::equal(rows, rows + nr, t->shape));
    };
    auto top_value = [&](const TensorP &t, int dt) {
        return !t || (t->dtype == dt && t->ndims == nr + 1 && std::equal(tops, tops + nr + 1, t->shape));
    };
    auto pair_value = [&](const TensorP &t) {
        return t->dtype == PT_FLOAT32 && t->ndims == nr + 1 && std::equal(rows, rows + nr, t->shape) && t->shape[nr] == 2;
    };
    if (!stats || !entropy || !pair_value(stats) || !row_value(entropy) || !row_value(g_logprob) || !row_value(g_entropy) ||
        !top_value(top_index, PT_INT32) || !top_value(g_top, PT_FLOAT32) || (g_top && !top_index)) {
        set_invalid("logProbs gradients need the forward pass's results and float32 upstream gradients of their shapes");
        return nullptr;
    }
    std::vector<TensorP> in = {a, tokens, stats, entropy};
    int given = 0;
    const TensorP *more[4] = {&top_index, &g_logprob, &g_entropy, &g_top};
    for (int i = 0; i < 4; i++)
        if (*more[i]) {
            in.push_back(*more[i]);
            given |= 1 << i;
        }
    if (fusion_active()) {
        NativeSpec sp;
        sp.kind = NAT_LOGPROBS_BACKWARD;
        sp.given = given;
        return fusion_record_native(sp, in, a->shape, a->ndims, a->dtype);
    }
    for (const TensorP &t : in)
        if (!guard(t)) return nullptr;
    TensorP out = output_tensor(a->shape, a->ndims, a->dtype);
    return out && logprobs_backward_run(in, given, out) ? out : nullptr;
}

// ------------------------------------------------------ steps of a plan
TensorP native_execute_model(const NativeSpec &sp, const std::vector<TensorP> &in)
{
    bool ok = false;
    TensorP out;
    switch (sp.kind) {
    case NAT_ATTENTION:
        out = output_tensor(in[0]->shape, in[0]->ndims, in[0]->dtype);
        ok = out && attention_run(in[0], in[1], in[2], sp.causal, sp.eps, sp.q_seq, sp.k_seq, out,
                                  in.size() > 3 ? in[3] : nullptr, in.size() > 4 ? in[4] : nullptr);
        break;
    case NAT_ATTENTION_BACKWARD: {
        const TensorP to[3] = {output_tensor(in[0]->shape, in[0]->ndims, in[0]->dtype), in[6], in[7]};
        out = to[0];
        const TensorP ops[7] = {in[0], in[1], in[2], in[3], in[4], in[5], in.size() > 8 ? in[8] : nullptr};
        ok = out && attention_backward_run(ops, sp.causal, sp.eps, sp.q_seq, sp.k_seq, to);
        break;
    }
    case NAT_LAYERNORM_BACKWARD: {
        size_t at = 2;
        const TensorP scale = sp.has_scale ? in[at++] : nullptr, bias = sp.has_bias ? in[at++] : nullptr;
        TensorP to[3] = {output_tensor(in[0]->shape, in[0]->ndims, in[0]->dtype), nullptr, nullptr};
        if (scale) to[1] = in[at++];
        if (bias) to[2] = in[at++];
        out = to[0];
        ok = out && layernorm_backward_run(in[0], in[1], sp.axes, sp.naxes, sp.eps, scale, bias, to);
        break;
    }
    case NAT_LOGPROBS: {
        TensorP to[5] = {output_tensor(in[1]->shape, in[1]->ndims, PT_FLOAT32)};
        for (size_t i = 2; i < in.size(); i++) to[i - 1] = in[i];
        out = to[0];
        ok = out && logprobs_run(in[0], in[1], sp.top, to);
        break;
    }
    case NAT_LOGPROBS_BACKWARD:
        out = output_tensor(in[0]->shape, in[0]->ndims, in[0]->dtype);
        ok = out && logprobs_backward_run(in, sp.given, out);
        break;
    default: set_runtime("Unknown native step");
    }
    return ok ? out : nullptr;
}

}  // namespace phpt
