// One AdamW step over many tensors in one launch (a few hundred tensors: a
// launch a hundred), for gfx950.  Per element, in this order and without
// contraction, as the composed step's operations round:
//   m = m0 b1 + g (1 - b1),  v = v0 b2 + (g g) (1 - b2)
//   p = p0 (1 - rate decay) - (m / c1) / (sqrt(v / c2) + eps) rate
// with c = 1 - b^t; an element whose gradient is NaN stays as it was.
// HBM-bound: everything is read once and written once.
//
// The moments (and float32 masters of 16-bit parameters) of all tensors lie in
// one array each, a tensor's from a multiple of 256 elements on; parameters
// and gradients are the tensors themselves.  A block takes 2048 elements of
// one tensor, found by bisection of the first blocks in the kernel's
// arguments; a thread 8 side by side, 16 bytes of a 16-bit tensor.
//
// Moments in 8 bits: 256 elements share the power of two 2^e that takes the
// largest of them into [128, 256): a change of scale then leaves values that
// it keeps in range as they are.  The first moment is held as a sign, 4 bits
// of exponent and 3 of mantissa, the root of the second (half the range) as 4
// and 4 bits.  Both are rounded up or down by 16 drawn bits with the
// probability of the distance: a second moment moves by 0.1 % a step, less
// than half a step of any 8-bit format, and would never decay if it went to
// the nearest.  An element one of whose new moments is NaN or 2^126 and more
// stays as it was: it would take its whole block along, or round up past
// float32.
#include "pt_common.h"

#include <algorithm>
#include <math.h>

namespace pt {

constexpr int kAdamTensors = 64;   // a launch: 3.4 KiB of arguments
constexpr int kAdamBlock = 2048;   // elements

struct AdamTensor {
    const void *p0, *g;
    void *p;
    long long n, at;        // elements, and where its moments begin
    unsigned first;         // block of the launch
    uint8_t pdt, gdt, decay;
};

struct AdamArgs {
    AdamTensor t[kAdamTensors];
    int count;
    const void *m0, *v0;
    void *m, *v;
    const float *master0;
    float *master;
    const int8_t *me0, *ve0;
    int8_t *me, *ve;
    const int32_t *draws0;
    int32_t *draws;
    const float *rate, *power1_0, *power2_0;
    float *power1, *power2;   // written by the first launch, else null
    float b1, one_b1, b2, one_b2, eps, decay, rate_value, decay_value;
};

typedef unsigned ad_u32x4 __attribute__((ext_vector_type(4), aligned(1)));
typedef unsigned ad_u32x2 __attribute__((ext_vector_type(2), aligned(1)));

template <int DT>
__device__ __forceinline__ void ad_load8(const void *base, long long i, float (&v)[8])
{
    using S = typename DType<DT>::S;
    const S *p = (const S *)base + i;
#pragma unroll
    for (int q = 0; q < 8 * (int)sizeof(S) / 16; q++) {
        union { ad_u32x4 raw; S s[16 / sizeof(S)]; } u;
        u.raw = __builtin_nontemporal_load((const ad_u32x4 *)(p + q * (16 / sizeof(S))));
#pragma unroll
        for (int k = 0; k < (int)(16 / sizeof(S)); k++) v[q * (16 / sizeof(S)) + k] = DType<DT>::to_c(u.s[k]);
    }
}

template <int DT>
__device__ __forceinline__ void ad_store8(void *base, long long i, const float (&v)[8])
{
    using S = typename DType<DT>::S;
    S *p = (S *)base + i;
#pragma unroll
    for (int q = 0; q < 8 * (int)sizeof(S) / 16; q++) {
        union { ad_u32x4 raw; S s[16 / sizeof(S)]; } u;
#pragma unroll
        for (int k = 0; k < (int)(16 / sizeof(S)); k++) u.s[k] = DType<DT>::from_c(v[q * (16 / sizeof(S)) + k]);
        __builtin_nontemporal_store(u.raw, (ad_u32x4 *)(p + q * (16 / sizeof(S))));
    }
}

// `live` of 8 elements from i on, of a tensor of dtype dt (uniform in a block)
template <int DT>
__device__ __forceinline__ void ad_load_as(const void *base, long long i, int live, float (&v)[8])
{
    if (live >= 8) return ad_load8<DT>(base, i, v);
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = k < live ? DType<DT>::to_c(((const typename DType<DT>::S *)base)[i + k]) : 0.0f;
}
__device__ __forceinline__ void ad_load(const void *base, int dt, long long i, int live, float (&v)[8])
{
    if (dt == PT_FLOAT32) ad_load_as<PT_FLOAT32>(base, i, live, v);
    else if (dt == PT_FLOAT16) ad_load_as<PT_FLOAT16>(base, i, live, v);
    else ad_load_as<PT_BFLOAT16>(base, i, live, v);
}
template <int DT>
__device__ __forceinline__ void ad_store_as(void *base, long long i, int live, const float (&v)[8])
{
    if (live >= 8) return ad_store8<DT>(base, i, v);
#pragma unroll
    for (int k = 0; k < 8; k++)
        if (k < live) ((typename DType<DT>::S *)base)[i + k] = DType<DT>::from_c(v[k]);
}
__device__ __forceinline__ void ad_store(void *base, int dt, long long i, int live, const float (&v)[8])
{
    if (dt == PT_FLOAT32) ad_store_as<PT_FLOAT32>(base, i, live, v);
    else if (dt == PT_FLOAT16) ad_store_as<PT_FLOAT16>(base, i, live, v);
    else ad_store_as<PT_BFLOAT16>(base, i, live, v);
}

// 32 bits spread over 32 bits: the finalizer of MurmurHash3 (A. Appleby)
__device__ __forceinline__ uint32_t ad_mix(uint32_t h)
{
    h ^= h >> 16;
    h *= 0x85EBCA6Bu;
    h ^= h >> 13;
    h *= 0xC2B2AE35u;
    return h ^ (h >> 16);
}

// 8-bit values.  A code's bits, moved to a float's exponent and mantissa,
// are its value times 2^-120 (its exponent bias is 7), below the least
// normal value too; the block's power of two is one more exact factor.
__device__ __forceinline__ float ad_power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
template <bool ROOT>
__device__ __forceinline__ float ad_decode(uint32_t code, float scale)
{
    const uint32_t bits = ROOT ? code << 19 : (code & 127u) << 20;
    const float x = __uint_as_float(bits) * 0x1p120f * scale;
    if constexpr (ROOT) return x * x;
    else return code & 128u ? -x : x;
}
// drawn: 16 bits
template <bool ROOT>
__device__ __forceinline__ uint32_t ad_encode(float x, float inverse, uint32_t drawn)
{
    constexpr int LOW = ROOT ? 19 : 20;
    const uint32_t size = __float_as_uint(fabsf(x) * inverse * 0x1p-120f);
    const uint32_t code = (size + (drawn << (LOW - 16)) + (1u << (LOW - 17))) >> LOW;
    return ROOT ? code : code | (x < 0.0f ? 128u : 0u);
}
// exponent of the power of two for a block's largest magnitude
__device__ __forceinline__ int ad_exponent(float top) { return max((int)(__float_as_uint(top) >> 23) - 127 - 7, -126); }
// the largest of 32 lanes' values (a block's 256 elements are 8 in each)
__device__ __forceinline__ float ad_top(float v)
{
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, PT_WAVE));
    return v;
}

template <bool SMALL, bool MASTER>
__global__ __launch_bounds__(256) void k_adamw(AdamArgs a)
{
    int lo = 0;
    for (int hi = a.count; hi - lo > 1;) {
        const int mid = (lo + hi) >> 1;
        if (a.t[mid].first <= blockIdx.x) lo = mid;
        else hi = mid;
    }
    const AdamTensor &t = a.t[lo];
    const float power1 = a.power1_0[0] * a.b1, power2 = a.power2_0[0] * a.b2;
    const float c1 = (power1 - 1.0f) * -1.0f, c2 = (power2 - 1.0f) * -1.0f;
    const float rate = a.rate ? a.rate[0] : a.rate_value;
    const float keep = a.rate ? (rate * a.decay - 1.0f) * -1.0f : a.decay_value;
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.power1) {
        *a.power1 = power1;
        *a.power2 = power2;
        if (SMALL) *a.draws = (int32_t)((uint32_t)*a.draws0 + 1u);
    }
    const long long i = (long long)(blockIdx.x - t.first) * kAdamBlock + threadIdx.x * 8;
    // (the block of 256 that holds the tensor's end is written whole; lanes
    // past it leave in the 32s that share one)
    if (i >= ((t.n + 255) & ~255ll)) return;
    const long long s = t.at + i;
    const int live = (int)max(0ll, min(8ll, t.n - i));
    float p[8], g[8], m[8], v[8];
    if constexpr (MASTER) ad_load8<PT_FLOAT32>(a.master0, s, p);
    else ad_load(t.p0, t.pdt, i, live, p);
    ad_load(t.g, t.gdt, i, live, g);
    float ms = 0.0f, vs = 0.0f;
    if constexpr (SMALL) {
        const ad_u32x2 mc = *(const ad_u32x2 *)((const uint8_t *)a.m0 + s), vc = *(const ad_u32x2 *)((const uint8_t *)a.v0 + s);
        ms = ad_power(a.me0[s >> 8]);
        vs = ad_power(a.ve0[s >> 8]);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            m[k] = ad_decode<false>(mc[k >> 2] >> (8 * (k & 3)) & 255u, ms);
            v[k] = ad_decode<true>(vc[k >> 2] >> (8 * (k & 3)) & 255u, vs);
        }
    } else {
        ad_load8<PT_FLOAT32>(a.m0, s, m);
        ad_load8<PT_FLOAT32>(a.v0, s, v);
    }
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const float mk = m[k] * a.b1 + g[k] * a.one_b1;
        const float vk = v[k] * a.b2 + (g[k] * g[k]) * a.one_b2;
        const float step = (mk / c1) / (sqrtf(vk / c2) + a.eps) * rate;
        const float pk = (t.decay ? p[k] * keep : p[k]) - step;
        const bool taken = k < live && (SMALL ? fabsf(mk) < 0x1p126f && vk < 0x1p126f : g[k] == g[k]);
        m[k] = taken ? mk : k < live ? m[k] : 0.0f;
        v[k] = taken ? vk : k < live ? v[k] : 0.0f;
        p[k] = taken ? pk : k < live ? p[k] : 0.0f;
    }
    if constexpr (MASTER) ad_store8<PT_FLOAT32>(a.master, s, p);
    ad_store(t.p, t.pdt, i, live, p);
    if constexpr (SMALL) {
        float mt = 0.0f, vt = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            v[k] = sqrtf(v[k]);
            mt = fmaxf(mt, fabsf(m[k]));
            vt = fmaxf(vt, v[k]);
        }
        const int me = ad_exponent(ad_top(mt)), ve = ad_exponent(ad_top(vt));
        const float mi = ad_power(-me), vi = ad_power(-ve);
        const uint32_t key = ad_mix((uint32_t)*a.draws0);
        ad_u32x2 mc = {0, 0}, vc = {0, 0};
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const uint32_t drawn = ad_mix((uint32_t)(s + k) + key + (uint32_t)(s >> 32) * 0x9E3779B9u);
            mc[k >> 2] |= ad_encode<false>(m[k], mi, drawn & 0xffffu) << (8 * (k & 3));
            vc[k >> 2] |= ad_encode<true>(v[k], vi, drawn >> 16) << (8 * (k & 3));
        }
        *(ad_u32x2 *)((uint8_t *)a.m + s) = mc;
        *(ad_u32x2 *)((uint8_t *)a.v + s) = vc;
        if ((threadIdx.x & 31) == 0) {
            a.me[s >> 8] = (int8_t)me;
            a.ve[s >> 8] = (int8_t)ve;
        }
    } else {
        ad_store8<PT_FLOAT32>(a.m, s, m);
        ad_store8<PT_FLOAT32>(a.v, s, v);
    }
}

// float32 values of 8-bit moments; n a multiple of 256
__global__ __launch_bounds__(256) void k_adamw_moments(const uint8_t *m, const int8_t *me, const uint8_t *v, const int8_t *ve,
                                                       float *mo, float *vo, long long n)
{
    for (long long s = ((long long)blockIdx.x * 256 + threadIdx.x) * 8; s < n; s += (long long)gridDim.x * 2048) {
        const ad_u32x2 mc = *(const ad_u32x2 *)(m + s), vc = *(const ad_u32x2 *)(v + s);
        const float ms = ad_power(me[s >> 8]), vs = ad_power(ve[s >> 8]);
        float x[8], y[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            x[k] = ad_decode<false>(mc[k >> 2] >> (8 * (k & 3)) & 255u, ms);
            y[k] = ad_decode<true>(vc[k >> 2] >> (8 * (k & 3)) & 255u, vs);
        }
        ad_store8<PT_FLOAT32>(mo, s, x);
        ad_store8<PT_FLOAT32>(vo, s, y);
    }
}

static bool adam_dtype(int dt) { return dt == PT_FLOAT32 || dt == PT_FLOAT16 || dt == PT_BFLOAT16; }

}  // namespace pt

using namespace pt;

extern "C" {

pt_status pt_adamw(const pt_adamw_desc *d, const pt_adamw_tensor *tensors, int count, pt_stream_t stream)
{
    if (!d || count < 0 || (count && !tensors)) return fail(PT_ERR_INVALID, "AdamW misses its description or tensors");
    if (d->bits != 32 && d->bits != 8) return fail(PT_ERR_INVALID, "AdamW moments have 32 or 8 bits");
    for (double b : {d->beta1, d->beta2})
        if (!(b >= 0.0 && b < 1.0)) return fail(PT_ERR_INVALID, "AdamW betas must be in [0, 1)");
    for (double x : {d->epsilon, d->weight_decay, d->rate ? 0.0 : d->rate_value})
        if (!(x >= 0.0) || !isfinite(x)) return fail(PT_ERR_INVALID, "AdamW epsilon, decay and rate must be finite and not negative");
    if (!d->first || !d->second || !d->new_first || !d->new_second || !d->power1 || !d->power2 || !d->new_power1 ||
        !d->new_power2 || !d->master != !d->new_master)
        return fail(PT_ERR_INVALID, "AdamW misses a state");
    if (d->bits == 8 && (!d->first_exponent || !d->second_exponent || !d->new_first_exponent || !d->new_second_exponent ||
                         !d->draws || !d->new_draws))
        return fail(PT_ERR_INVALID, "AdamW misses a state of 8-bit moments");
    size_t at = 0;
    for (int i = 0; i < count; i++) {
        const pt_adamw_tensor &t = tensors[i];
        if (t.n > ((size_t)1 << 40)) return fail(PT_ERR_INVALID, "AdamW tensor too large");
        if (t.n && ((!t.param && !d->master) || !t.grad || !t.new_param))
            return fail(PT_ERR_INVALID, "AdamW tensor misses an address");
        if (!adam_dtype(t.param_dtype) || !adam_dtype(t.grad_dtype))
            return fail(PT_ERR_INVALID, "AdamW takes float32, float16 or bfloat16 parameters and gradients");
        if (t.at % 256 || t.at < at) return fail(PT_ERR_INVALID, "AdamW moments lie in the tensors' order, from multiples of 256 on");
        at = t.at + t.n;
    }
    PT_TRY(ensure_init());
    AdamArgs a = {};
    a.m0 = d->first;
    a.v0 = d->second;
    a.m = d->new_first;
    a.v = d->new_second;
    a.master0 = d->master;
    a.master = d->new_master;
    a.me0 = d->first_exponent;
    a.ve0 = d->second_exponent;
    a.me = d->new_first_exponent;
    a.ve = d->new_second_exponent;
    a.draws0 = d->draws;
    a.draws = d->new_draws;
    a.rate = d->rate;
    a.power1_0 = d->power1;
    a.power2_0 = d->power2;
    a.power1 = d->new_power1;
    a.power2 = d->new_power2;
    a.b1 = (float)d->beta1;
    a.one_b1 = (float)(1.0 - d->beta1);
    a.b2 = (float)d->beta2;
    a.one_b2 = (float)(1.0 - d->beta2);
    a.eps = (float)d->epsilon;
    a.decay = (float)d->weight_decay;
    a.rate_value = (float)d->rate_value;
    a.decay_value = (float)(1.0 - d->rate_value * d->weight_decay);
    hipStream_t s = stream_of(stream);
    auto launch = [&](unsigned blocks) {
        if (d->bits == 8) {
            if (d->master) k_adamw<true, true><<<blocks, 256, 0, s>>>(a);
            else k_adamw<true, false><<<blocks, 256, 0, s>>>(a);
        } else {
            if (d->master) k_adamw<false, true><<<blocks, 256, 0, s>>>(a);
            else k_adamw<false, false><<<blocks, 256, 0, s>>>(a);
        }
        a.power1 = a.power2 = nullptr;
    };
    long long blocks = 0;
    bool launched = false;
    for (int i = 0; i < count; i++) {
        const pt_adamw_tensor &t = tensors[i];
        if (!t.n) continue;
        const long long more = ((long long)t.n + kAdamBlock - 1) / kAdamBlock;
        if (a.count == kAdamTensors || blocks + more > 0x7fffffff) {
            launch((unsigned)blocks);
            a.count = 0;
            blocks = 0;
            launched = true;
        }
        AdamTensor &to = a.t[a.count++];
        to = {t.param, t.grad, t.new_param, (long long)t.n, (long long)t.at, (unsigned)blocks, (uint8_t)t.param_dtype,
              (uint8_t)t.grad_dtype, (uint8_t)(t.decay && d->weight_decay > 0.0)};
        blocks += more;
    }
    if (!blocks && !launched) {
        // no element: the powers go on all the same
        a.t[0] = {};
        a.count = 1;
        blocks = 1;
    }
    if (blocks) launch((unsigned)blocks);
    return check_hip(hipGetLastError(), "AdamW");
}

pt_status pt_adamw_moments(const void *first, const int8_t *first_exponent, const void *second, const int8_t *second_exponent,
                           float *first_values, float *second_values, size_t n, pt_stream_t stream)
{
    if (n % 256 || n > ((size_t)1 << 48)) return fail(PT_ERR_INVALID, "8-bit moments come in blocks of 256 elements");
    if (n && (!first || !first_exponent || !second || !second_exponent || !first_values || !second_values))
        return fail(PT_ERR_INVALID, "8-bit moments miss an operand");
    PT_TRY(ensure_init());
    if (!n) return PT_OK;
    const unsigned blocks = (unsigned)std::min<size_t>((n + 2047) / 2048, 1 << 20);
    k_adamw_moments<<<blocks, 256, 0, stream_of(stream)>>>((const uint8_t *)first, first_exponent, (const uint8_t *)second,
                                                           second_exponent, first_values, second_values, (long long)n);
    return check_hip(hipGetLastError(), "8-bit moments");
}

}  // extern "C"
