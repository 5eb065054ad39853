// Dispatch of the operators around a block's matrix products: the rotation
// of queries and keys, the gated projection, and the AdamW step over many
// tensors.  As in
// model_ops.cpp, each checks its operands, allocates its results and
// launches through the C-ABI, or records one native step in a Fusion scope.
#include "runtime.hpp"

#include <limits.h>
#include <math.h>
#include <string.h>

#include <algorithm>

namespace phpt {

// ----------------------------------------------------------------- rotary
RotaryP make_rotary(int part, double base, bool interleaved, double factor, double context, double low, double high,
                    double magnitude, const double *frequencies)
{
    if (part < 2 || part % 2 || part > 256) {
        set_invalid("Rotary turns an even number of 2 to 256 elements");
        return nullptr;
    }
    if (!frequencies && (!(base > 0.0) || !isfinite(base))) {
        set_invalid("Rotary base must be finite and positive");
        return nullptr;
    }
    if (!(factor > 0.0) || !isfinite(factor) || !(context >= 0.0) || !isfinite(context)) {
        set_invalid("Rotary factor must be finite and positive, its context not negative");
        return nullptr;
    }
    if (!isfinite(low) || !isfinite(high) || low >= high) {
        set_invalid("Rotary needs fewer turns for low than for high");
        return nullptr;
    }
    if (!isfinite((float)magnitude)) {
        set_invalid("Rotary magnitude must be finite");
        return nullptr;
    }
    auto r = std::make_shared<Rotary>();
    r->part = part;
    r->interleaved = interleaved;
    r->magnitude = magnitude;
    std::vector<double> turns;
    for (int i = 0; i < part / 2; i++) {
        double f = frequencies ? frequencies[i] : pow(base, -2.0 * i / part);
        if (!isfinite(f)) {
            set_invalid("Rotary frequencies must be finite");
            return nullptr;
        }
        if (factor != 1.0 && context == 0.0) f /= factor;
        if (factor != 1.0 && context > 0.0) {
            // what turns often within the context stays, what turns seldom is stretched
            const double keep = std::min(1.0, std::max(0.0, (context * fabs(f) / (2.0 * M_PI) - low) / (high - low)));
            f = f * keep + f / factor * (1.0 - keep);
        }
        turns.push_back(f / (2.0 * M_PI));
    }
    const int shape[1] = {part / 2};
    r->turns = from_host(turns.data(), shape, 1, PT_FLOAT64);
    return r->turns ? r : nullptr;
}

// Checks that need no device, and the description without addresses.
static bool rotary_desc(const TensorP &q, const TensorP &k, const TensorP &positions, const RotaryP &plan, const TensorP &qs,
                        const TensorP &ks, double eps, pt_rotary_desc &d)
{
    if (!q || !plan) {
        set_invalid("Missing tensor operand");
        return false;
    }
    const int nd = q->ndims;
    if (!low_or_f32(q->dtype) || (k && k->dtype != q->dtype)) {
        set_invalid("rotary requires matching float32, float16 or bfloat16 heads");
        return false;
    }
    if ((nd != 3 && nd != 4) || (k && (k->ndims != nd || !std::equal(q->shape, q->shape + nd - 2, k->shape) ||
                                       k->shape[nd - 1] != q->shape[nd - 1]))) {
        set_invalid("rotary requires [tokens, heads, size] or [sequences, tokens, heads, size], queries and keys of the "
                    "same tokens and size");
        return false;
    }
    const int size = q->shape[nd - 1];
    if (size > 256 || plan->part > size) {
        set_invalid("rotary heads have at most 256 elements, and no fewer than are turned");
        return false;
    }
    if (q->shape[nd - 2] > 65536 || (k && k->shape[nd - 2] > 65536)) {
        set_invalid("rotary takes at most 65536 heads");
        return false;
    }
    const long long rows = (nd == 4 ? (long long)q->shape[0] : 1ll) * q->shape[nd - 3];
    if (rows > INT_MAX) {
        set_invalid("rotary takes at most %d tokens", INT_MAX);
        return false;
    }
    if (positions) {
        const bool each = positions->ndims == nd - 2 && std::equal(q->shape, q->shape + nd - 2, positions->shape);
        const bool common = nd == 4 && positions->ndims == 1 && positions->shape[0] == q->shape[1];
        if (positions->dtype != PT_INT32 || (!each && !common)) {
            set_invalid("rotary positions must be int32, one for each token");
            return false;
        }
    }
    for (const TensorP *s : {&qs, &ks})
        if (*s && ((*s)->dtype != q->dtype || (*s)->ndims != 1 || (*s)->shape[0] != size)) {
            set_invalid("rotary scales must have a head's size and the heads' dtype");
            return false;
        }
    if (ks && !k) {
        set_invalid("rotary has a scale for keys but no keys");
        return false;
    }
    if (!(eps > 0.0) || !isfinite((float)eps) || (float)eps <= 0.0f) {
        set_invalid("rotary epsilon must be finite and greater than zero");
        return false;
    }
    memset(&d, 0, sizeof(d));
    d.dtype = q->dtype;
    d.sequences = nd == 4 ? q->shape[0] : 1;
    d.tokens = q->shape[nd - 3];
    d.heads[0] = q->shape[nd - 2];
    d.heads[1] = k ? k->shape[nd - 2] : 0;
    d.size = size;
    d.part = plan->part;
    d.interleaved = plan->interleaved;
    d.magnitude = plan->magnitude;
    d.epsilon = eps;
    d.turns = (const double *)plan->turns->data();
    return true;
}

static void rotary_positions(const TensorP &positions, const TensorP &q, pt_rotary_desc &d)
{
    if (!positions) return;
    d.positions = (const int32_t *)positions->data();
    d.position_strides[0] = q->ndims == 4 && positions->ndims == 2 ? positions->strides[0] : 0;
    d.position_strides[1] = positions->strides[positions->ndims - 1];
}

static bool rotary_run(const TensorP &q, const TensorP &k, const TensorP &positions, const RotaryP &plan, const TensorP &qs,
                       const TensorP &ks, double eps, const TensorP out[2])
{
    pt_rotary_desc d;
    if (!rotary_desc(q, k, positions, plan, qs, ks, eps, d)) return false;
    rotary_positions(positions, q, d);
    TensorP a = head_operand(q, d.strides[0]), b = k ? head_operand(k, d.strides[1]) : nullptr;
    TensorP sa = qs ? materialize(qs) : nullptr, sb = ks ? materialize(ks) : nullptr;
    if (!a || (k && !b) || (qs && !sa) || (ks && !sb)) return false;
    const void *x[2] = {a->data(), b ? b->data() : nullptr}, *s[2] = {sa ? sa->data() : nullptr, sb ? sb->data() : nullptr};
    void *y[2] = {out[0]->data(), k ? out[1]->data() : nullptr};
    return check_status(pt_rotary(&d, x, s, y, nullptr), "Rotary kernel failed");
}

// Which optional operands of a native step are there (NativeSpec.given), and
// their order behind q.
enum { ROT_K = 1, ROT_POSITIONS = 2, ROT_QS = 4, ROT_KS = 8, ROT_GQ = 16, ROT_GK = 32 };

bool cuda_array_rotary(const TensorP &q, const TensorP &k, const TensorP &positions, const RotaryP &plan, const TensorP &qs,
                       const TensorP &ks, double eps, TensorP out[2])
{
    pt_rotary_desc d;
    if (!rotary_desc(q, k, positions, plan, qs, ks, eps, d)) return false;
    out[1] = nullptr;
    if (fusion_active()) {
        NativeSpec sp;
        sp.kind = NAT_ROTARY;
        sp.eps = eps;
        sp.rotary = plan;
        std::vector<TensorP> ins = {q};
        const TensorP *more[4] = {&k, &positions, &qs, &ks};
        for (int i = 0; i < 4; i++)
            if (*more[i]) {
                ins.push_back(*more[i]);
                sp.given |= 1 << i;
            }
        TensorP box = k ? record_buffer(k->shape, k->ndims, k->dtype) : nullptr;
        if (k && !box) return false;
        if (box) ins.push_back(box);
        out[0] = fusion_record_native(sp, ins, q->shape, q->ndims, q->dtype);
        if (out[0] && box) out[1] = record_result(box, out[0]);
        return out[0] && (!k || out[1]);
    }
    for (const TensorP *t : {&q, &k, &positions, &qs, &ks})
        if (*t && !guard(*t)) return false;
    out[0] = output_tensor(q->shape, q->ndims, q->dtype);
    if (out[0] && k) out[1] = make_empty(k->shape, k->ndims, k->dtype);
    if (!out[0] || (k && !out[1])) return false;
    return rotary_run(q, k, positions, plan, qs, ks, eps, out);
}

static bool rotary_backward_run(const TensorP &q, const TensorP &k, const TensorP &positions, const RotaryP &plan,
                                const TensorP &qs, const TensorP &ks, double eps, const TensorP &gq, const TensorP &gk,
                                const TensorP *out)
{
    pt_rotary_desc d;
    if (!rotary_desc(q, k, positions, plan, qs, ks, eps, d)) return false;
    rotary_positions(positions, q, d);
    TensorP a = head_operand(q, d.strides[0]), b = k ? head_operand(k, d.strides[1]) : nullptr;
    TensorP sa = qs ? materialize(qs) : nullptr, sb = ks ? materialize(ks) : nullptr;
    TensorP ga = gq ? materialize(gq) : nullptr, gb = gk ? materialize(gk) : nullptr;
    if (!a || (k && !b) || (qs && !sa) || (ks && !sb) || (gq && !ga) || (gk && !gb)) return false;
    if (!gq) d.heads[0] = 0;
    if (!gk) d.heads[1] = 0;
    auto at = [](const TensorP &t) -> void * { return t ? t->data() : nullptr; };
    const void *x[2] = {at(a), at(b)}, *s[2] = {at(sa), at(sb)}, *g[2] = {at(ga), at(gb)};
    void *dx[2] = {at(out[0]), at(out[1])}, *ds[2] = {gq ? at(out[2]) : nullptr, gk ? at(out[3]) : nullptr};
    return check_status(pt_rotary_backward(&d, x, s, g, (ga ? ga : gb)->dtype, dx, ds, nullptr), "Rotary gradient kernel failed");
}

bool cuda_array_rotary_backward(const TensorP &q, const TensorP &k, const TensorP &positions, const RotaryP &plan,
                                const TensorP &qs, const TensorP &ks, double eps, const TensorP &gq, const TensorP &gk,
                                TensorP out[4])
{
    pt_rotary_desc d;
    if (!rotary_desc(q, k, positions, plan, qs, ks, eps, d)) return false;
    auto fits = [&](const TensorP &g, const TensorP &x) {
        return !g || (x && same_shape(*g, *x) && (g->dtype == q->dtype || g->dtype == PT_FLOAT32));
    };
    if ((!gq && !gk) || !fits(gq, q) || !fits(gk, k) || (gq && gk && gq->dtype != gk->dtype)) {
        set_invalid("rotary's upstream gradients must have the outputs' shapes, in float32 or their dtype");
        return false;
    }
    // what a side without an upstream gradient would get does not exist
    const TensorP want[4] = {gq ? q : nullptr, gk ? k : nullptr, gq ? qs : nullptr, gk ? ks : nullptr};
    const int first = gq ? 0 : 1;
    for (int i = 0; i < 4; i++) out[i] = nullptr;
    if (fusion_active()) {
        NativeSpec sp;
        sp.kind = NAT_ROTARY_BACKWARD;
        sp.eps = eps;
        sp.rotary = plan;
        std::vector<TensorP> ins = {q};
        const TensorP *more[6] = {&k, &positions, &qs, &ks, &gq, &gk};
        for (int i = 0; i < 6; i++)
            if (*more[i]) {
                ins.push_back(*more[i]);
                sp.given |= 1 << i;
            }
        TensorP box[4];
        for (int i = first + 1; i < 4; i++)
            if (want[i]) {
                box[i] = record_buffer(want[i]->shape, want[i]->ndims, want[i]->dtype);
                if (!box[i]) return false;
                ins.push_back(box[i]);
            }
        out[first] = fusion_record_native(sp, ins, want[first]->shape, want[first]->ndims, want[first]->dtype);
        if (!out[first]) return false;
        for (int i = first + 1; i < 4; i++)
            if (box[i] && !(out[i] = record_result(box[i], out[first]))) return false;
        return true;
    }
    for (const TensorP *t : {&q, &k, &positions, &qs, &ks, &gq, &gk})
        if (*t && !guard(*t)) return false;
    for (int i = first; i < 4; i++)
        if (want[i]) {
            out[i] = i == first ? output_tensor(want[i]->shape, want[i]->ndims, want[i]->dtype)
                                : make_empty(want[i]->shape, want[i]->ndims, want[i]->dtype);
            if (!out[i]) return false;
        }
    return rotary_backward_run(q, k, positions, plan, qs, ks, eps, gq, gk, out);
}

// -------------------------------------------------------- gated projection
static bool gated_desc(const TensorP &x, const TensorP &gate, const TensorP &up, int activation, pt_gated_desc &d)
{
    if (!x || !gate || !up) {
        set_invalid("Missing tensor operand");
        return false;
    }
    if (!low_or_f32(x->dtype) || gate->dtype != x->dtype || up->dtype != x->dtype) {
        set_invalid("gatedProjection requires matching float32, float16 or bfloat16 operands");
        return false;
    }
    if (x->ndims < 1 || gate->ndims != 2 || !same_shape(*gate, *up) || gate->shape[0] != x->shape[x->ndims - 1]) {
        set_invalid("gatedProjection requires [.., inner] and two matrices [inner, outer] of one shape");
        return false;
    }
    if (activation < PT_GATE_SILU || activation > PT_GATE_SIGMOID) {
        set_invalid("gatedProjection activations are silu, gelu, relu and sigmoid");
        return false;
    }
    long long rows = 1;
    bool none = false;
    for (int i = 0; i + 1 < x->ndims; i++) none = none || !x->shape[i];
    for (int i = 0; !none && i + 1 < x->ndims && rows <= 1 << 21; i++) rows *= x->shape[i];
    if (none) rows = 0;
    if (rows > 1 << 21 || gate->shape[0] > 1 << 21 || gate->shape[1] > 1 << 21) {
        set_invalid("gatedProjection takes at most %d rows, and elements in each", 1 << 21);
        return false;
    }
    memset(&d, 0, sizeof(d));
    d.dtype = x->dtype;
    d.activation = activation;
    d.rows = (int)rows;
    d.inner = gate->shape[0];
    d.outer = gate->shape[1];
    return true;
}

static int gated_shape(const Tensor &x, const Tensor &gate, int *shape)
{
    std::copy(x.shape, x.shape + x.ndims, shape);
    shape[x.ndims - 1] = gate.shape[1];
    return x.ndims;
}

// what pt_gated keeps of both products, in bytes an element
static int kept_bytes(const TensorP &x) { return x->dtype == PT_FLOAT32 ? 8 : 6; }

static bool gated_run(const TensorP &x, const TensorP &gate, const TensorP &up, int activation, const TensorP &h,
                      const TensorP &kept)
{
    pt_gated_desc d;
    if (!gated_desc(x, gate, up, activation, d)) return false;
    TensorP a = materialize(x), b = materialize(gate), c = materialize(up);
    if (!a || !b || !c) return false;
    return check_status(pt_gated(&d, a->data(), b->data(), c->data(), h->data(), kept ? kept->data() : nullptr, nullptr),
                        "Gated projection kernel failed");
}

bool cuda_array_gated(const TensorP &x, const TensorP &gate, const TensorP &up, int activation, bool keep, TensorP out[2])
{
    pt_gated_desc d;
    if (!gated_desc(x, gate, up, activation, d)) return false;
    int shape[kMaxDims];
    const int nd = gated_shape(*x, *gate, shape), both[3] = {kept_bytes(x), d.rows, d.outer};
    out[1] = nullptr;
    if (fusion_active()) {
        NativeSpec sp;
        sp.kind = NAT_GATED;
        sp.activation = activation;
        std::vector<TensorP> ins = {x, gate, up};
        TensorP box = keep ? record_buffer(both, 3, PT_UINT8) : nullptr;
        if (keep && !box) return false;
        if (box) ins.push_back(box);
        out[0] = fusion_record_native(sp, ins, shape, nd, x->dtype);
        if (out[0] && box) out[1] = record_result(box, out[0]);
        return out[0] && (!keep || out[1]);
    }
    if (!guard(x) || !guard(gate) || !guard(up)) return false;
    out[0] = output_tensor(shape, nd, x->dtype);
    if (out[0] && keep) out[1] = make_empty(both, 3, PT_UINT8);
    if (!out[0] || (keep && !out[1])) return false;
    return gated_run(x, gate, up, activation, out[0], out[1]);
}

static bool gated_backward_run(const TensorP &x, const TensorP &gate, const TensorP &up, const TensorP &kept,
                               const TensorP &grad, int activation, const TensorP *out)
{
    pt_gated_desc d;
    if (!gated_desc(x, gate, up, activation, d)) return false;
    TensorP a = materialize(x), b = materialize(gate), c = materialize(up), k = materialize(kept), g = materialize(grad);
    if (!a || !b || !c || !k || !g) return false;
    auto at = [](const TensorP &t) -> void * { return t ? t->data() : nullptr; };
    return check_status(pt_gated_backward(&d, a->data(), b->data(), c->data(), k->data(), g->data(), g->dtype, at(out[0]),
                                          at(out[1]), at(out[2]), nullptr),
                        "Gated projection gradient kernel failed");
}

// Results in order; the first of those wanted is the native step's own.
enum { GATED_X = 1, GATED_WEIGHTS = 2 };

bool cuda_array_gated_backward(const TensorP &x, const TensorP &gate, const TensorP &up, const TensorP &kept,
                               const TensorP &grad, int activation, bool want_x, bool want_weights, TensorP out[3])
{
    pt_gated_desc d;
    if (!gated_desc(x, gate, up, activation, d)) return false;
    int shape[kMaxDims];
    const int nd = gated_shape(*x, *gate, shape);
    if (!kept || kept->dtype != PT_UINT8 || kept->ndims != 3 || kept->shape[0] != kept_bytes(x) || kept->shape[1] != d.rows ||
        kept->shape[2] != d.outer) {
        set_invalid("gatedProjection gradients need the forward pass's products");
        return false;
    }
    if (!grad || grad->ndims != nd || !std::equal(shape, shape + nd, grad->shape) ||
        (grad->dtype != x->dtype && grad->dtype != PT_FLOAT32)) {
        set_invalid("gatedProjection's upstream gradient must have the output's shape, in float32 or its dtype");
        return false;
    }
    if (!want_x && !want_weights) {
        set_invalid("gatedProjection gradients: none is wanted");
        return false;
    }
    const TensorP want[3] = {want_x ? x : nullptr, want_weights ? gate : nullptr, want_weights ? up : nullptr};
    const int first = want_x ? 0 : 1;
    for (int i = 0; i < 3; i++) out[i] = nullptr;
    if (fusion_active()) {
        NativeSpec sp;
        sp.kind = NAT_GATED_BACKWARD;
        sp.activation = activation;
        sp.given = (want_x ? GATED_X : 0) | (want_weights ? GATED_WEIGHTS : 0);
        std::vector<TensorP> ins = {x, gate, up, kept, grad};
        TensorP box[3];
        for (int i = first + 1; i < 3; i++)
            if (want[i]) {
                box[i] = record_buffer(want[i]->shape, want[i]->ndims, want[i]->dtype);
                if (!box[i]) return false;
                ins.push_back(box[i]);
            }
        out[first] = fusion_record_native(sp, ins, want[first]->shape, want[first]->ndims, x->dtype);
        if (!out[first]) return false;
        for (int i = first + 1; i < 3; i++)
            if (box[i] && !(out[i] = record_result(box[i], out[first]))) return false;
        return true;
    }
    for (const TensorP *t : {&x, &gate, &up, &kept, &grad})
        if (!guard(*t)) return false;
    for (int i = first; i < 3; i++)
        if (want[i]) {
            out[i] = i == first ? output_tensor(want[i]->shape, want[i]->ndims, want[i]->dtype)
                                : make_empty(want[i]->shape, want[i]->ndims, want[i]->dtype);
            if (!out[i]) return false;
        }
    return gated_backward_run(x, gate, up, kept, grad, activation, out);
}

// ------------------------------------------------------------------ AdamW
static constexpr long long kMomentBlock = 256;  // elements that share an exponent

// Where each tensor's moments begin; the arrays' size, or -1.
static long long adamw_places(const std::vector<TensorP> &params, std::vector<size_t> &at)
{
    long long total = 0;
    for (const TensorP &p : params) {
        at.push_back((size_t)total);
        total += ((long long)p->numel() + kMomentBlock - 1) / kMomentBlock * kMomentBlock;
        if (total / kMomentBlock > INT_MAX) return -1;
    }
    return total;
}

long long adamw_blocks(const std::vector<TensorP> &params)
{
    std::vector<size_t> at;
    const long long total = adamw_places(params, at);
    return total < 0 ? -1 : total / kMomentBlock;
}

static bool adamw_check(const AdamwStepP &step, const std::vector<TensorP> &params, const std::vector<TensorP> &grads,
                        const std::vector<TensorP> &states, const TensorP &rate)
{
    if (params.empty() || params.size() != grads.size() || (int)params.size() != step->count() ||
        (int)states.size() != step->states()) {
        set_invalid("AdamW needs parameters, as many gradients and decay flags, and a state");
        return false;
    }
    for (size_t i = 0; i < params.size(); i++) {
        if (!params[i] || !grads[i]) {
            set_invalid("Missing tensor operand");
            return false;
        }
        if (!low_or_f32(params[i]->dtype) || !low_or_f32(grads[i]->dtype)) {
            set_invalid("AdamW over many tensors takes float32, float16 or bfloat16 parameters and gradients");
            return false;
        }
        if (!same_shape(*params[i], *grads[i])) {
            set_invalid("Each gradient must have the same shape as its parameter");
            return false;
        }
    }
    std::vector<size_t> at;
    const long long total = adamw_places(params, at);
    if (total < 0) {
        set_invalid("AdamW's parameters have too many elements together");
        return false;
    }
    auto fits = [&](const TensorP &t, int dtype, long long n) {
        return t && t->dtype == dtype && t->ndims == 1 && t->shape[0] == n;
    };
    auto blocks = [&](const TensorP &t, int dtype) {
        return t && t->dtype == dtype && t->ndims == 2 && t->shape[0] == total / kMomentBlock && t->shape[1] == kMomentBlock;
    };
    const int moment = step->bits == 8 ? PT_UINT8 : PT_FLOAT32;
    bool ok = blocks(states[0], moment) && blocks(states[1], moment) && fits(states[2], PT_FLOAT32, 1) &&
              fits(states[3], PT_FLOAT32, 1);
    size_t k = 4;
    if (step->master) ok = ok && blocks(states[k++], PT_FLOAT32);
    if (step->bits == 8)
        ok = ok && fits(states[k], PT_INT8, total / kMomentBlock) && fits(states[k + 1], PT_INT8, total / kMomentBlock) &&
             fits(states[k + 2], PT_INT32, 1);
    if (!ok) {
        set_invalid("AdamW's state does not belong to these parameters");
        return false;
    }
    if (rate && !fits(rate, PT_FLOAT32, 1)) {
        set_invalid("A learning rate on the device must be float32 [1]");
        return false;
    }
    return true;
}

static bool adamw_run(const AdamwStep &step, const std::vector<TensorP> &params, const std::vector<TensorP> &grads,
                      const std::vector<TensorP> &states, const TensorP &rate, const std::vector<TensorP> &out)
{
    std::vector<size_t> at;
    adamw_places(params, at);
    std::vector<TensorP> held;  // packed operands
    auto packed = [&](const TensorP &t) -> const void * {
        TensorP u = materialize(t);
        if (!u) return nullptr;
        held.push_back(u);
        return u->data();
    };
    std::vector<pt_adamw_tensor> table(params.size());
    for (size_t i = 0; i < params.size(); i++) {
        pt_adamw_tensor &t = table[i];
        t.n = params[i]->numel();
        t.at = at[i];
        t.param_dtype = params[i]->dtype;
        t.grad_dtype = grads[i]->dtype;
        t.decay = step.decay[i];
        t.new_param = out[i]->data();
        t.param = packed(params[i]);
        t.grad = packed(grads[i]);
        if (t.n && (!t.param || !t.grad)) return false;
    }
    pt_adamw_desc d;
    memset(&d, 0, sizeof(d));
    d.bits = step.bits;
    d.beta1 = step.beta1;
    d.beta2 = step.beta2;
    d.epsilon = step.epsilon;
    d.weight_decay = step.weight_decay;
    d.rate_value = step.rate;
    const void *s[8];
    void *n[8];
    for (size_t i = 0; i < states.size(); i++) {
        s[i] = packed(states[i]);
        n[i] = out[params.size() + i]->data();
        if (!s[i]) return false;
    }
    if (rate && !(d.rate = (const float *)packed(rate))) return false;
    d.first = s[0];
    d.second = s[1];
    d.power1 = (const float *)s[2];
    d.power2 = (const float *)s[3];
    d.new_first = n[0];
    d.new_second = n[1];
    d.new_power1 = (float *)n[2];
    d.new_power2 = (float *)n[3];
    size_t k = 4;
    if (step.master) {
        d.master = (const float *)s[k];
        d.new_master = (float *)n[k++];
    }
    if (step.bits == 8) {
        d.first_exponent = (const int8_t *)s[k];
        d.second_exponent = (const int8_t *)s[k + 1];
        d.draws = (const int32_t *)s[k + 2];
        d.new_first_exponent = (int8_t *)n[k];
        d.new_second_exponent = (int8_t *)n[k + 1];
        d.new_draws = (int32_t *)n[k + 2];
    }
    return check_status(pt_adamw(&d, table.data(), (int)table.size(), nullptr), "AdamW kernel failed");
}

bool cuda_array_adamw(const AdamwStepP &step, const std::vector<TensorP> &params, const std::vector<TensorP> &grads,
                      const std::vector<TensorP> &states, const TensorP &rate, std::vector<TensorP> &out)
{
    if (!adamw_check(step, params, grads, states, rate)) return false;
    std::vector<TensorP> like = params;
    like.insert(like.end(), states.begin(), states.end());
    std::vector<TensorP> ins = params;
    ins.insert(ins.end(), grads.begin(), grads.end());
    ins.insert(ins.end(), states.begin(), states.end());
    if (rate) ins.push_back(rate);
    out.clear();
    if (fusion_active()) {
        NativeSpec sp;
        sp.kind = NAT_ADAMW;
        sp.adamw = step;
        std::vector<TensorP> boxes;
        for (size_t i = 1; i < like.size(); i++) {
            boxes.push_back(record_buffer(like[i]->shape, like[i]->ndims, like[i]->dtype));
            if (!boxes.back()) return false;
        }
        ins.insert(ins.end(), boxes.begin(), boxes.end());
        out.push_back(fusion_record_native(sp, ins, like[0]->shape, like[0]->ndims, like[0]->dtype));
        if (!out[0]) return false;
        for (const TensorP &b : boxes) {
            out.push_back(record_result(b, out[0]));
            if (!out.back()) return false;
        }
        return true;
    }
    for (const TensorP &t : ins)
        if (!guard(t)) return false;
    for (size_t i = 0; i < like.size(); i++) {
        out.push_back(i ? make_empty(like[i]->shape, like[i]->ndims, like[i]->dtype)
                        : output_tensor(like[i]->shape, like[i]->ndims, like[i]->dtype));
        if (!out.back()) return false;
    }
    return adamw_run(*step, params, grads, states, rate, out);
}

TensorP cuda_array_adamw_masters(const std::vector<TensorP> &params)
{
    if (fusion_active()) {
        set_invalid("AdamW's state is made outside of a Fusion scope");
        return nullptr;
    }
    for (const TensorP &p : params) {
        if (!guard(p)) return nullptr;
        if (!low_or_f32(p->dtype)) {
            set_invalid("AdamW over many tensors takes float32, float16 or bfloat16 parameters and gradients");
            return nullptr;
        }
    }
    std::vector<size_t> at;
    const long long total = adamw_places(params, at);
    if (total < 0) {
        set_invalid("AdamW's parameters have too many elements together");
        return nullptr;
    }
    const int shape[2] = {(int)(total / kMomentBlock), (int)kMomentBlock};
    TensorP out = full(shape, 2, PT_FLOAT32, scalar_from_double(0.0));
    if (!out) return nullptr;
    for (size_t i = 0; i < params.size(); i++) {
        const Tensor &p = *params[i];
        if (p.numel() && !check_status(pt_cast(p.storage->ptr, p.dtype, p.strides, p.offset, (float *)out->data() + at[i],
                                               PT_FLOAT32, p.shape, p.ndims, nullptr),
                                       "AdamW masters"))
            return nullptr;
    }
    return out;
}

static bool moments_run(const TensorP *in, const TensorP *out)
{
    TensorP t[4];
    for (int i = 0; i < 4; i++)
        if (!(t[i] = materialize(in[i]))) return false;
    return check_status(pt_adamw_moments(t[0]->data(), (const int8_t *)t[1]->data(), t[2]->data(), (const int8_t *)t[3]->data(),
                                         (float *)out[0]->data(), (float *)out[1]->data(), t[0]->numel(), nullptr),
                        "Moments kernel failed");
}

bool cuda_array_adamw_moments(const TensorP &first, const TensorP &first_exponent, const TensorP &second,
                              const TensorP &second_exponent, TensorP out[2])
{
    auto codes = [&](const TensorP &t) {
        return t && t->dtype == PT_UINT8 && t->ndims == 2 && t->shape[1] == kMomentBlock && t->shape[0] == first->shape[0];
    };
    auto exponents = [&](const TensorP &t) {
        return t && t->dtype == PT_INT8 && t->ndims == 1 && t->shape[0] == first->shape[0];
    };
    if (!codes(first) || !codes(second) || !exponents(first_exponent) || !exponents(second_exponent)) {
        set_invalid("8-bit moments are uint8 [blocks, %d], with an int8 exponent a block", (int)kMomentBlock);
        return false;
    }
    const std::vector<TensorP> in = {first, first_exponent, second, second_exponent};
    if (fusion_active()) {
        NativeSpec sp;
        sp.kind = NAT_ADAMW_MOMENTS;
        TensorP box = record_buffer(first->shape, 2, PT_FLOAT32);
        if (!box) return false;
        out[0] = fusion_record_native(sp, {first, first_exponent, second, second_exponent, box}, first->shape, 2, PT_FLOAT32);
        return out[0] && (out[1] = record_result(box, out[0]));
    }
    for (const TensorP &t : in)
        if (!guard(t)) return false;
    out[0] = output_tensor(first->shape, 2, PT_FLOAT32);
    out[1] = make_empty(first->shape, 2, PT_FLOAT32);
    return out[0] && out[1] && moments_run(in.data(), out);
}

// ------------------------------------------------------ steps of a plan
TensorP native_execute_block(const NativeSpec &sp, const std::vector<TensorP> &in)
{
    bool ok = false;
    TensorP out;
    size_t at = 1;
    auto next = [&](int bit) { return sp.given & bit ? in[at++] : TensorP(); };
    switch (sp.kind) {
    case NAT_ROTARY: {
        const TensorP k = next(ROT_K), positions = next(ROT_POSITIONS), qs = next(ROT_QS), ks = next(ROT_KS);
        const TensorP to[2] = {output_tensor(in[0]->shape, in[0]->ndims, in[0]->dtype), k ? in[at] : nullptr};
        out = to[0];
        ok = out && rotary_run(in[0], k, positions, sp.rotary, qs, ks, sp.eps, to);
        break;
    }
    case NAT_ROTARY_BACKWARD: {
        const TensorP k = next(ROT_K), positions = next(ROT_POSITIONS), qs = next(ROT_QS), ks = next(ROT_KS);
        const TensorP gq = next(ROT_GQ), gk = next(ROT_GK), &first = gq ? in[0] : k;
        TensorP to[4];
        out = output_tensor(first->shape, first->ndims, first->dtype);
        to[gq ? 0 : 1] = out;
        if (gq && gk) to[1] = in[at++];
        if (gq && qs) to[2] = in[at++];
        if (gk && ks) to[3] = in[at++];
        ok = out && rotary_backward_run(in[0], k, positions, sp.rotary, qs, ks, sp.eps, gq, gk, to);
        break;
    }
    case NAT_GATED: {
        int shape[kMaxDims];
        const int nd = gated_shape(*in[0], *in[1], shape);
        out = output_tensor(shape, nd, in[0]->dtype);
        ok = out && gated_run(in[0], in[1], in[2], sp.activation, out, in.size() > 3 ? in[3] : nullptr);
        break;
    }
    case NAT_GATED_BACKWARD: {
        const TensorP &first = sp.given & GATED_X ? in[0] : in[1];
        out = output_tensor(first->shape, first->ndims, first->dtype);
        TensorP to[3];
        at = 5;
        to[sp.given & GATED_X ? 0 : 1] = out;
        if ((sp.given & GATED_X) && (sp.given & GATED_WEIGHTS)) to[1] = in[at++];
        if (sp.given & GATED_WEIGHTS) to[2] = in[at++];
        ok = out && gated_backward_run(in[0], in[1], in[2], in[3], in[4], sp.activation, to);
        break;
    }
    case NAT_ADAMW: {
        const size_t n = (size_t)sp.adamw->count(), states = (size_t)sp.adamw->states();
        auto part = [&](size_t from, size_t count) { return std::vector<TensorP>(in.begin() + from, in.begin() + from + count); };
        size_t k = 2 * n + states;
        const TensorP rate = sp.adamw->has_rate ? in[k++] : nullptr;
        std::vector<TensorP> to = {output_tensor(in[0]->shape, in[0]->ndims, in[0]->dtype)};
        to.insert(to.end(), in.begin() + k, in.end());
        out = to[0];
        ok = out && adamw_run(*sp.adamw, part(0, n), part(n, n), part(2 * n, states), rate, to);
        break;
    }
    case NAT_ADAMW_MOMENTS: {
        const TensorP to[2] = {output_tensor(in[0]->shape, 2, PT_FLOAT32), in[4]};
        out = to[0];
        ok = out && moments_run(in.data(), to);
        break;
    }
    default: set_runtime("Unknown native step");
    }
    return ok ? out : nullptr;
}

}  // namespace phpt
