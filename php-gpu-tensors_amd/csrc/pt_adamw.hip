// One AdamW step over many tensors in one launch (more than 64: a launch for
// each 64), for gfx950.  Per element, in this order and without
// contraction, as the composed step's operations round:
//   m = m0 b1 + g (1 - b1),  v = v0 b2 + (g g) (1 - b2)
//   p = p0 (1 - rate decay) - (m / c1) / (sqrt(v / c2) + eps) rate
// with c = 1 - b^t; an element whose gradient is NaN stays as it was.
// HBM-bound: everything is read once and written once.  134 M elements,
// bfloat16 with float32 masters: 626-664 us, 5.7-6.0 TB/s (a large copy 5.0).
// With moments in 8 bits and no masters 382-419 us for a third of the bytes:
// 100 vector instructions an element, of which the exact root and the drawn
// numbers are half, take longer than HBM.
//
// The moments (and float32 masters of 16-bit parameters) of all tensors lie in
// one array each, a tensor's from a multiple of 256 elements on; parameters
// and gradients are the tensors themselves.  A block takes 2048 elements of
// one tensor, found by bisection of the first blocks in the kernel's
// arguments, its waves 256 side by side, twice.
//
// Moments in 8 bits: 256 elements share the power of two 2^e that takes the
// largest of them into [128, 256): a change of scale then leaves values that
// it keeps in range as they are.  The first moment is held as a sign, 4 bits
// of exponent and 3 of mantissa, the root of the second (half the range) as 4
// and 4 bits.  Both are rounded up or down by 16 drawn bits with the
// probability of the distance: a second moment moves by 0.1 % a step, less
// than half a step of any 8-bit format, and would never decay if it went to
// the nearest.  A root whose first moment is not held as zero is not held as
// zero either, but as the smallest value at least: otherwise an element whose
// gradients are 1e-6 of its block's largest would now and then step by its
// first moment over epsilon, hundreds of rates.  An element one of whose new moments is NaN or 2^126 and more
// stays as it was: it would take its whole block along, or round up past
// float32.
#include "pt_common.h"

#include <algorithm>
#include <math.h>

namespace pt {

constexpr int kAdamTensors = 64;   // of a launch, in its arguments
constexpr int kAdamRounds = 2;     // 256 elements that a wave takes at once
constexpr int kAdamBlock = 4 * kAdamRounds * 256;  // elements
constexpr long long kAdamMost = kLaunchThreads / 256;  // blocks of a launch
constexpr long long kAdamPart = 1ll << 31;             // elements of a tensor that a launch's table takes as one

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
static_assert(sizeof(AdamArgs) <= 4096, "a kernel's arguments hold the table");

// A thread's 4 elements side by side, in 2, 4 or 1 words.
typedef unsigned ad_u32x4 __attribute__((ext_vector_type(4), aligned(1)));
typedef unsigned ad_u32x2 __attribute__((ext_vector_type(2), aligned(1)));

template <int DT>
__device__ __forceinline__ void ad_load4(const void *base, long long i, float (&v)[4])
{
    if constexpr (DT == PT_FLOAT32) {
        const ad_u32x4 w = __builtin_nontemporal_load((const ad_u32x4 *)((const float *)base + i));
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = __uint_as_float(w[k]);
    } else {
        const ad_u32x2 w = __builtin_nontemporal_load((const ad_u32x2 *)((const uint16_t *)base + i));
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = DType<DT>::to_c((uint16_t)(w[k / 2] >> (k & 1 ? 16 : 0)));
    }
}

template <int DT>
__device__ __forceinline__ void ad_store4(void *base, long long i, const float (&v)[4])
{
    if constexpr (DT == PT_FLOAT32) {
        const ad_u32x4 w = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        __builtin_nontemporal_store(w, (ad_u32x4 *)((float *)base + i));
    } else {
        const ad_u32x2 w = {pack_low<DT>(v[0], v[1]), pack_low<DT>(v[2], v[3])};
        __builtin_nontemporal_store(w, (ad_u32x2 *)((uint16_t *)base + i));
    }
}

// `live` of 4 elements from i on, of a tensor of dtype dt (uniform in a block)
template <int DT>
__device__ __forceinline__ void ad_load_as(const void *base, long long i, int live, float (&v)[4])
{
    if (live >= 4) return ad_load4<DT>(base, i, v);
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = k < live ? DType<DT>::to_c(((const typename DType<DT>::S *)base)[i + k]) : 0.0f;
}
__device__ __forceinline__ void ad_load(const void *base, int dt, long long i, int live, float (&v)[4])
{
    if (dt == PT_FLOAT32) ad_load_as<PT_FLOAT32>(base, i, live, v);
    else if (dt == PT_FLOAT16) ad_load_as<PT_FLOAT16>(base, i, live, v);
    else ad_load_as<PT_BFLOAT16>(base, i, live, v);
}
template <int DT>
__device__ __forceinline__ void ad_store_as(void *base, long long i, int live, const float (&v)[4])
{
    if (live >= 4) return ad_store4<DT>(base, i, v);
#pragma unroll
    for (int k = 0; k < 4; k++)
        if (k < live) ((typename DType<DT>::S *)base)[i + k] = DType<DT>::from_c(v[k]);
}
__device__ __forceinline__ void ad_store(void *base, int dt, long long i, int live, const float (&v)[4])
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
// (v_ldexp_f32 takes all of it in one instruction, rounding once)
template <bool ROOT>
__device__ __forceinline__ float ad_decode(uint32_t code, int e)
{
    if constexpr (ROOT) return ldexpf(__uint_as_float(code << 19), 120 + e);
    else return ldexpf(__uint_as_float((code & 127u) << 20 | (code & 128u) << 24), 120 + e);
}
// drawn: 16 bits
template <bool ROOT>
__device__ __forceinline__ uint32_t ad_encode(float x, int e, uint32_t drawn)
{
    constexpr int LOW = ROOT ? 19 : 20;
    const uint32_t size = __float_as_uint(ldexpf(fabsf(x), -120 - e));
    const uint32_t code = (size + (drawn << (LOW - 16)) + (1u << (LOW - 17))) >> LOW;
    return ROOT ? code : code | (x < 0.0f ? 128u : 0u);
}
// exponent of the power of two for a block's largest magnitude
__device__ __forceinline__ int ad_exponent(float top) { return max((int)(__float_as_uint(top) >> 23) - 127 - 7, -126); }

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
    // 8 bits: m / c1 / (sqrt(v) / sqrt(c2) + eps) rate
    const float small_rate = rate / c1, small_root = 1.0f / sqrtf(c2);
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.power1) {
        *a.power1 = power1;
        *a.power2 = power2;
        if (SMALL) *a.draws = (int32_t)((uint32_t)*a.draws0 + 1u);
    }
    // a wave takes 256 elements at a time, an 8-bit block, 4 a lane; it
    // writes the 256 that hold the tensor's end whole
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const long long i0 = (long long)(blockIdx.x - t.first) * kAdamBlock + wave * (kAdamRounds * 256);
    const int rounds = (int)min((long long)kAdamRounds, (t.n - i0 + 255) >> 8);  // (may be negative)
    const uint32_t key = SMALL ? ad_mix((uint32_t)*a.draws0) : 0;
    // elements that are left of the tensor (uniform), and of a lane's 4
    auto rest = [&](int r) { return (int)min(256ll, t.n - i0 - r * 256); };
    float p[kAdamRounds][4], g[kAdamRounds][4], m[kAdamRounds][4], v[kAdamRounds][4];
    uint32_t mc[kAdamRounds], vc[kAdamRounds];
    int me[kAdamRounds], ve[kAdamRounds];
#pragma unroll
    for (int r = 0; r < kAdamRounds; r++) {
        if (r >= rounds) break;
        const long long i = i0 + r * 256 + lane * 4, s = t.at + i;
        const int live = max(0, min(4, rest(r) - lane * 4));
        if constexpr (MASTER) ad_load4<PT_FLOAT32>(a.master0, s, p[r]);
        else ad_load(t.p0, t.pdt, i, live, p[r]);
        ad_load(t.g, t.gdt, i, live, g[r]);
        if constexpr (SMALL) {
            mc[r] = __builtin_nontemporal_load((const uint32_t *)((const uint8_t *)a.m0 + s));
            vc[r] = __builtin_nontemporal_load((const uint32_t *)((const uint8_t *)a.v0 + s));
            me[r] = a.me0[(t.at + i0) / 256 + r];
            ve[r] = a.ve0[(t.at + i0) / 256 + r];
        } else {
            ad_load4<PT_FLOAT32>(a.m0, s, m[r]);
            ad_load4<PT_FLOAT32>(a.v0, s, v[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < kAdamRounds; r++) {
        if (r >= rounds) break;
        const long long i = i0 + r * 256 + lane * 4, s = t.at + i;
        // (nothing to ask of each element where all 256 are there: 426 -> 409 us for 134 M in 8 bits)
        auto round = [&](auto WHOLE) {
            constexpr bool whole = decltype(WHOLE)::value;
            const int live = whole ? 4 : max(0, min(4, rest(r) - lane * 4));
            float root[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if constexpr (SMALL) {
                    m[r][k] = ad_decode<false>(mc[r] >> (8 * k) & 255u, me[r]);
                    root[k] = ad_decode<true>(vc[r] >> (8 * k) & 255u, ve[r]);
                    v[r][k] = root[k] * root[k];  // (exact: 10 bits)
                }
                const float gk = g[r][k];
                const float mk = m[r][k] * a.b1 + gk * a.one_b1;
                const float vk = v[r][k] * a.b2 + (gk * gk) * a.one_b2;
                float step, new_root = 0.0f;
                if constexpr (SMALL) {
                    // the root that is held serves the step too, and the divisions
                    // by numbers of the whole call are products: a few ulps of the step
                    new_root = sqrtf(vk);
                    step = mk * small_rate * __builtin_amdgcn_rcpf(new_root * small_root + a.eps);
                } else {
                    step = (mk / c1) / (sqrtf(vk / c2) + a.eps) * rate;
                }
                const float pk = (t.decay ? p[r][k] * keep : p[r][k]) - step;
                const bool taken = k < live && (SMALL ? fabsf(mk) < 0x1p126f && vk < 0x1p126f : gk == gk);
                if constexpr (SMALL) root[k] = taken ? new_root : k < live ? root[k] : 0.0f;
                else v[r][k] = taken ? vk : k < live ? v[r][k] : 0.0f;
                m[r][k] = taken ? mk : k < live ? m[r][k] : 0.0f;
                p[r][k] = taken ? pk : k < live ? p[r][k] : 0.0f;
            }
            if constexpr (MASTER) ad_store4<PT_FLOAT32>(a.master, s, p[r]);
            ad_store(t.p, t.pdt, i, live, p[r]);
            if constexpr (SMALL) {
                float mt = 0.0f, vt = 0.0f;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    mt = fmaxf(mt, fabsf(m[r][k]));
                    vt = fmaxf(vt, root[k]);
                }
                const int mx = ad_exponent(wave_all(mt, FMax{})), vx = ad_exponent(wave_all(vt, FMax{}));
                uint32_t mo = 0, vo = 0;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t drawn = ad_mix((uint32_t)(s + k) + key + (uint32_t)(s >> 32) * 0x9E3779B9u);
                    const uint32_t code = ad_encode<false>(m[r][k], mx, drawn & 0xffffu);
                    mo |= code << (8 * k);
                    vo |= max(ad_encode<true>(root[k], vx, drawn >> 16), min(code & 127u, 1u)) << (8 * k);
                }
                __builtin_nontemporal_store(mo, (uint32_t *)((uint8_t *)a.m + s));
                __builtin_nontemporal_store(vo, (uint32_t *)((uint8_t *)a.v + s));
                if (lane == 0) {
                    a.me[(t.at + i0) / 256 + r] = (int8_t)mx;
                    a.ve[(t.at + i0) / 256 + r] = (int8_t)vx;
                }
            } else {
                ad_store4<PT_FLOAT32>(a.m, s, m[r]);
                ad_store4<PT_FLOAT32>(a.v, s, v[r]);
            }
        };
        if (rest(r) == 256) round(std::true_type{});
        else round(std::false_type{});
    }
}

// float32 values of 8-bit moments; a wave takes blocks of 256, 4 elements a lane
__global__ __launch_bounds__(256) void k_adamw_moments(const uint8_t *m, const int8_t *me, const uint8_t *v, const int8_t *ve,
                                                       float *mo, float *vo, long long blocks)
{
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    for (long long b = (long long)blockIdx.x * 4 + wave; b < blocks; b += (long long)gridDim.x * 4) {
        const long long s = b * 256 + lane * 4;
        const uint32_t mc = __builtin_nontemporal_load((const uint32_t *)(m + s)), vc = __builtin_nontemporal_load((const uint32_t *)(v + s));
        const int mx = me[b], vx = ve[b];
        float x[4], y[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            x[k] = ad_decode<false>(mc >> (8 * k) & 255u, mx);
            const float root = ad_decode<true>(vc >> (8 * k) & 255u, vx);
            y[k] = root * root;
        }
        ad_store4<PT_FLOAT32>(mo, s, x);
        ad_store4<PT_FLOAT32>(vo, s, y);
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
    // (every block reads them, one writes them)
    if (d->new_power1 == d->power1 || d->new_power2 == d->power2 || (d->bits == 8 && d->new_draws == d->draws))
        return fail(PT_ERR_INVALID, "AdamW's new powers and draws must not take the old ones' place");
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
    if (d->bits == 8) a.eps = std::max(a.eps, 0x1p-126f);  // (the reciprocal of less is infinite, of a first moment of 0 too)
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
        for (long long from = 0; from < (long long)t.n; from += kAdamPart) {
            const long long n = std::min((long long)t.n - from, kAdamPart), more = (n + kAdamBlock - 1) / kAdamBlock;
            if (a.count == kAdamTensors || blocks + more > kAdamMost) {
                launch((unsigned)blocks);
                a.count = 0;
                blocks = 0;
                launched = true;
            }
            auto part = [&](const void *base, int dtype) { return base ? (const char *)base + from * (long long)dtype_size(dtype) : nullptr; };
            AdamTensor &to = a.t[a.count++];
            to = {part(t.param, t.param_dtype), part(t.grad, t.grad_dtype), (void *)part(t.new_param, t.param_dtype), n,
                  (long long)t.at + from, (unsigned)blocks, (uint8_t)t.param_dtype, (uint8_t)t.grad_dtype,
                  (uint8_t)(t.decay && d->weight_decay > 0.0)};
            blocks += more;
        }
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
    const unsigned blocks = launch_blocks((n / 256 + 3) / 4);
    k_adamw_moments<<<blocks, 256, 0, stream_of(stream)>>>((const uint8_t *)first, first_exponent, (const uint8_t *)second,
                                                           second_exponent, first_values, second_values, (long long)(n / 256));
    return check_hip(hipGetLastError(), "8-bit moments");
}

}  // extern "C"
