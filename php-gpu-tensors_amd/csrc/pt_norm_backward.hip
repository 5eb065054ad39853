// Gradients of layerNorm for gfx950.  With the row's mean and r = 1 /
// sqrt(variance + eps), x' = (x - mean) r, the upstream gradient g and
// h = g gamma:
//   dx     = r (h - mean(h) - x' mean(h x'))
//   dgamma = sum over rows of g x',   dbeta = sum over rows of g
// The statistics are recomputed from x, which has to be read anyway, so the
// forward pass keeps nothing.  HBM-bound: x and g are read once and dx is
// written once.  A walking block holds one row (or one a group of waves) in
// registers and adds its columns' part of dgamma and dbeta there over all
// the rows it takes; each block then writes one partial row of both, and a
// second kernel adds the partial rows in a fixed order, so results do not
// depend on timing.  8192 rows of 4096 float32: 80 us (5.0 TB/s) and 5 us;
// 6000 rows of 1001 bfloat16: 16 and 4 us.  Rows past 4096 elements take 16
// waves: chunks of two or four a thread, with the next row's beside them,
// spilled (4096 rows of 10001 bfloat16 256 us, 129 with 16 waves).
#include "pt_common.h"

#include <algorithm>
#include <math.h>

namespace pt {

typedef unsigned int nb_u32x4 __attribute__((ext_vector_type(4), aligned(1)));

// V elements from p, widened to fp32; 16 bytes at any element boundary
// (gfx950 loads them at every byte address).
template <int DT, int V, bool NT>
__device__ __forceinline__ void nb_load(const typename DType<DT>::S *p, float (&v)[V])
{
    using S = typename DType<DT>::S;
    constexpr int PK = 16 / sizeof(S);
    static_assert(V % PK == 0, "whole packs");
#pragma unroll
    for (int q = 0; q < V / PK; q++) {
        union { nb_u32x4 raw; S s[PK]; } u;
        if constexpr (NT) u.raw = __builtin_nontemporal_load((const nb_u32x4 *)(p + q * PK));
        else u.raw = *(const nb_u32x4 *)(p + q * PK);
#pragma unroll
        for (int i = 0; i < PK; i++) v[q * PK + i] = DType<DT>::to_c(u.s[i]);
    }
}

template <int DT, int V>
__device__ __forceinline__ void nb_store(typename DType<DT>::S *p, const float (&v)[V])
{
    using S = typename DType<DT>::S;
    constexpr int PK = 16 / sizeof(S);
#pragma unroll
    for (int q = 0; q < V / PK; q++) {
        union { nb_u32x4 raw; S s[PK]; } u;
#pragma unroll
        for (int i = 0; i < PK; i++) u.s[i] = DType<DT>::from_c(v[q * PK + i]);
        __builtin_nontemporal_store(u.raw, (nb_u32x4 *)(p + q * PK));
    }
}

struct NormBwdArgs {
    const void *x;
    const float *g;
    const void *gamma;   // null: ones
    void *dx;            // null: not wanted
    float *partial;      // [block][2][n]; null: no parameter gradients wanted
    long long rows;
    int n;
    float eps;
};

// fp32 statistics, rows of up to 64 * WPR * V * NCH elements, WPR waves a
// row and 8 / WPR rows at a time in a block of 8 waves (WPR 16: of 16).  V is 8 elements: one
// 16-byte load of x in 16 bits, two in 32.  A row that ends inside a chunk
// reads its last chunk V elements before the end; the elements that another
// lane owns count for nothing in the sums and get the same dx twice.
template <int DT, int PDT, int NCH, int WPR>
__global__ __launch_bounds__(64 * (WPR > 8 ? WPR : 8)) void k_norm_backward(NormBwdArgs a)
{
    using S = typename DType<DT>::S;
    using PS = typename DType<PDT>::S;
    constexpr int V = 8, W = WPR > 8 ? WPR : 8, RPB = W / WPR, TPR = 64 * WPR;
    __shared__ float lds[2][W][3];
    __shared__ float sums[WPR < 8 ? 2 * TPR * V * NCH : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = threadIdx.x % TPR, first = wave - wave % WPR;
    const int n = a.n;

    int at[NCH], skip[NCH];  // where the chunk is read, and how many of its elements another lane owns
    float gamma[NCH][V], dg[NCH][V], db[NCH][V];
#pragma unroll
    for (int c = 0; c < NCH; c++) {
        const int i = (c * TPR + t) * V;
        at[c] = min(i, n - V);  // rows of fewer than V elements have the kernels below
        skip[c] = min(V, i - at[c]);
        if (a.gamma) nb_load<PDT, V, false>((const PS *)a.gamma + at[c], gamma[c]);
#pragma unroll
        for (int k = 0; k < V; k++) {
            if (!a.gamma) gamma[c][k] = 1.0f;
            dg[c][k] = db[c][k] = 0.0f;
        }
    }
    auto load = [&](long long row, float (&x)[NCH][V], float (&g)[NCH][V]) {
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            if (skip[c] >= V) {  // past the row's end
#pragma unroll
                for (int k = 0; k < V; k++) x[c][k] = g[c][k] = 0.0f;
                continue;
            }
            nb_load<DT, V, true>((const S *)a.x + row * n + at[c], x[c]);
            nb_load<PT_FLOAT32, V, true>(a.g + row * n + at[c], g[c]);
        }
    };
    // sums over the row of up to three values, the same in every thread of it
    int turn = 0;
    auto row_sums = [&](float &p, float &q, float &r) {
        p = wave_all(p, FAdd{});
        q = wave_all(q, FAdd{});
        r = wave_all(r, FAdd{});
        if constexpr (WPR > 1) {
            float(&box)[W][3] = lds[turn];  // two in turn: one barrier a call keeps reads and writes apart
            turn ^= 1;
            if (lane == 0) {
                box[wave][0] = p;
                box[wave][1] = q;
                box[wave][2] = r;
            }
            __syncthreads();
            p = box[first][0];
            q = box[first][1];
            r = box[first][2];
#pragma unroll
            for (int w = 1; w < WPR; w++) {
                p += box[first + w][0];
                q += box[first + w][1];
                r += box[first + w][2];
            }
        }
    };
    const float inv_n = 1.0f / (float)n;
    auto process = [&](long long row, float (&x)[NCH][V], float (&g)[NCH][V], bool live) {
        float s = 0.0f, none = 0.0f, none2 = 0.0f;
#pragma unroll
        for (int c = 0; c < NCH; c++)
#pragma unroll
            for (int k = 0; k < V; k++) s += k >= skip[c] ? x[c][k] : 0.0f;
        row_sums(s, none, none2);
        const float mean = s * inv_n;
        float q = 0.0f, h1 = 0.0f, h2 = 0.0f;
#pragma unroll
        for (int c = 0; c < NCH; c++)
#pragma unroll
            for (int k = 0; k < V; k++) {
                const float d = x[c][k] - mean, h = g[c][k] * gamma[c][k];
                x[c][k] = d;
                if (k >= skip[c]) {
                    q = fmaf(d, d, q);
                    h1 += h;
                    h2 = fmaf(h, d, h2);
                }
            }
        row_sums(q, h1, h2);
        const float r = 1.0f / sqrtf(q * inv_n + a.eps);
        h1 *= inv_n;
        h2 *= inv_n * r;
        if (!live) return;
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            if (skip[c] >= V) continue;
            float out[V];
#pragma unroll
            for (int k = 0; k < V; k++) {
                const float u = x[c][k] * r, gk = g[c][k];
                out[k] = r * (gk * gamma[c][k] - h1 - u * h2);
                const float own = k >= skip[c] ? gk : 0.0f;
                dg[c][k] = fmaf(own, u, dg[c][k]);
                db[c][k] += own;
            }
            if (!a.dx) continue;
            nb_store<DT, V>((S *)a.dx + row * n + at[c], out);
        }
    };
    // rows blockIdx.x * RPB + wave / WPR and so on; the next row's loads are
    // issued before this row's reductions where registers hold two rows.
    // Every row group of a block runs the same number of turns, for the
    // barriers.
    const long long step = (long long)gridDim.x * RPB, row0 = (long long)blockIdx.x * RPB;
    const long long mine = wave / WPR;
    float x[NCH][V], g[NCH][V];
    auto clamp_row = [&](long long r) { return min(r, a.rows - 1); };
    if constexpr (NCH > 1) {
        for (long long r = row0; r < a.rows; r += step) {
            load(clamp_row(r + mine), x, g);
            process(r + mine, x, g, r + mine < a.rows);
        }
    }
    float xn[NCH][V], gn[NCH][V];
    if (NCH == 1 && row0 < a.rows) load(clamp_row(row0 + mine), x, g);
    for (long long r = row0; NCH == 1 && r < a.rows; r += step) {
        if (r + step < a.rows) load(clamp_row(r + step + mine), xn, gn);
        process(r + mine, x, g, r + mine < a.rows);
#pragma unroll
        for (int c = 0; c < NCH; c++)
#pragma unroll
            for (int k = 0; k < V; k++) {
                x[c][k] = xn[c][k];
                g[c][k] = gn[c][k];
            }
    }
    if (!a.partial) return;
    if constexpr (WPR < 8) {
        // the block's row groups add up in LDS, one after the other
        for (int w = 0; w < RPB; w++) {
            __syncthreads();
            if (wave / WPR != w) continue;
#pragma unroll
            for (int c = 0; c < NCH; c++)
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const int i = ((c * V + k) * TPR + t) * 2;
                    sums[i] = dg[c][k] = (w ? sums[i] : 0.0f) + dg[c][k];
                    sums[i + 1] = db[c][k] = (w ? sums[i + 1] : 0.0f) + db[c][k];
                }
        }
        if (wave / WPR != RPB - 1) return;
    }
    float *part = a.partial + (long long)blockIdx.x * 2 * n;
#pragma unroll
    for (int c = 0; c < NCH; c++)
#pragma unroll
        for (int k = 0; k < V; k++)
            if (k >= skip[c] && at[c] + k < n) {
                part[at[c] + k] = dg[c][k];
                part[n + at[c] + k] = db[c][k];
            }
}

// dgamma and dbeta from the partial rows: 64 columns a block, its 16 waves
// add a sixteenth of the partial rows each, in order, then the first adds
// the 16 sums.
template <int PDT, typename CT>
__global__ __launch_bounds__(1024) void k_norm_params(const CT *partial, int parts, int n, void *dgamma, void *dbeta)
{
    __shared__ CT box[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (int)blockIdx.x * 64 + lane;
    void *out = blockIdx.y ? dbeta : dgamma;
    if (!out) return;  // whole block
    CT s = 0;
    if (c < n) {
        const CT *p = partial + (long long)blockIdx.y * n + c;
#pragma unroll 8
        for (int r = wave; r < parts; r += 16) s += p[(long long)r * 2 * n];
    }
    box[wave][lane] = s;
    __syncthreads();
    if (wave || c >= n) return;
    for (int w = 1; w < 16; w++) s += box[w][lane];
    if constexpr (PDT == PT_FLOAT64) ((double *)out)[c] = s;
    else ((typename DType<PDT>::S *)out)[c] = DType<PDT>::from_c((float)s);
}

// Any other rows: fewer than 8 elements, more than 16384, or float64.  One
// block a row reads it three times (the later times from cache) and leaves
// mean and r for the columns' sums, which walk the rows once more.
template <int DT, typename CT>
__device__ __forceinline__ CT nb_value(const void *p, long long i)
{
    return (CT)DType<DT>::to_c(((const typename DType<DT>::S *)p)[i]);
}

template <typename CT>
__device__ __forceinline__ CT nb_block_sum(CT v, CT *box)
{
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, PT_WAVE);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) box[threadIdx.x >> 6] = v;
    __syncthreads();
    return box[0] + box[1] + box[2] + box[3];
}

template <int DT, int PDT, typename CT>
__global__ __launch_bounds__(256) void k_norm_backward_row(const void *x, const CT *g, const void *gamma, void *dx,
                                                           CT *stats, long long rows, int n, CT eps)
{
    __shared__ CT box[4];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const long long base = row * n;
        CT s = 0;
        for (int i = threadIdx.x; i < n; i += 256) s += nb_value<DT, CT>(x, base + i);
        const CT mean = nb_block_sum(s, box) / (CT)n;
        CT q = 0, h1 = 0, h2 = 0;
        for (int i = threadIdx.x; i < n; i += 256) {
            const CT d = nb_value<DT, CT>(x, base + i) - mean;
            const CT h = gamma ? g[base + i] * nb_value<PDT, CT>(gamma, i) : g[base + i];
            q += d * d;
            h1 += h;
            h2 += h * d;
        }
        q = nb_block_sum(q, box);
        h1 = nb_block_sum(h1, box) / (CT)n;
        const CT r = (CT)1 / (sizeof(CT) == 8 ? (CT)sqrt((double)(q / (CT)n + eps)) : (CT)sqrtf((float)(q / (CT)n + eps)));
        h2 = nb_block_sum(h2, box) / (CT)n * r;
        if (stats && threadIdx.x == 0) {
            stats[2 * row] = mean;
            stats[2 * row + 1] = r;
        }
        if (!dx) continue;
        for (int i = threadIdx.x; i < n; i += 256) {
            const CT u = (nb_value<DT, CT>(x, base + i) - mean) * r;
            const CT h = gamma ? g[base + i] * nb_value<PDT, CT>(gamma, i) : g[base + i];
            ((typename DType<DT>::S *)dx)[base + i] = DType<DT>::from_c((typename DType<DT>::C)(r * (h - h1 - u * h2)));
        }
    }
}

template <int DT, typename CT>
__global__ __launch_bounds__(256) void k_norm_backward_columns(const void *x, const CT *g, const CT *stats, CT *partial,
                                                               long long rows, int n)
{
    const int c = (int)blockIdx.x * 256 + threadIdx.x;
    if (c >= n) return;
    CT dg = 0, db = 0;
    for (long long r = blockIdx.y; r < rows; r += gridDim.y) {
        const CT gv = g[r * n + c];
        dg += gv * ((nb_value<DT, CT>(x, r * n + c) - stats[2 * r]) * stats[2 * r + 1]);
        db += gv;
    }
    partial[(long long)blockIdx.y * 2 * n + c] = dg;
    partial[(long long)blockIdx.y * 2 * n + n + c] = db;
}

template <int DT, int PDT, typename CT>
static pt_status norm_backward_general(const void *x, const void *g, const void *gamma, void *dx, void *dgamma,
                                       void *dbeta, long long rows, int n, CT eps, hipStream_t s)
{
    const bool params = dgamma || dbeta;
    const int parts = (int)std::min<long long>(rows, std::max(1, 2048 / ((n + 255) / 256)));
    void *scratch = nullptr;
    if (params) PT_TRY(scratch_alloc(&scratch, ((size_t)rows * 2 + (size_t)parts * 2 * n) * sizeof(CT), s));
    CT *stats = (CT *)scratch, *partial = stats ? stats + rows * 2 : nullptr;
    k_norm_backward_row<DT, PDT, CT><<<(unsigned)std::min(rows, 1ll << 20), 256, 0, s>>>(x, (const CT *)g, gamma, dx, stats,
                                                                                     rows, n, eps);
    if (params) {
        k_norm_backward_columns<DT, CT><<<dim3((n + 255) / 256, parts), 256, 0, s>>>(x, (const CT *)g, stats, partial, rows, n);
        k_norm_params<PDT, CT><<<dim3((n + 63) / 64, 2), 1024, 0, s>>>(partial, parts, n, dgamma, dbeta);
    }
    const pt_status st = check_hip(hipGetLastError(), "layerNorm gradient");
    if (scratch) scratch_free(scratch, s);
    return st;
}

template <int DT, int PDT>
static pt_status norm_backward_f32(NormBwdArgs a, void *dgamma, void *dbeta, hipStream_t s)
{
    if (a.n < 8 || a.n > 16384)
        return norm_backward_general<DT, PDT, float>(a.x, a.g, a.gamma, a.dx, dgamma, dbeta, a.rows, a.n, a.eps, s);
    const int wpr = a.n <= 512 ? 1 : a.n <= 1024 ? 2 : a.n <= 2048 ? 4 : 8, rpb = 8 / wpr;
    // two blocks a CU hide each other's reductions (one of 16 waves fills it)
    const int blocks = (int)std::min<long long>((a.rows + rpb - 1) / rpb, a.n <= 4096 ? 512 : 256);
    void *scratch = nullptr;
    if (dgamma || dbeta) PT_TRY(scratch_alloc(&scratch, (size_t)blocks * 2 * a.n * sizeof(float), s));
    a.partial = (float *)scratch;
    switch (wpr) {
    case 1: k_norm_backward<DT, PDT, 1, 1><<<blocks, 512, 0, s>>>(a); break;
    case 2: k_norm_backward<DT, PDT, 1, 2><<<blocks, 512, 0, s>>>(a); break;
    case 4: k_norm_backward<DT, PDT, 1, 4><<<blocks, 512, 0, s>>>(a); break;
    default:
        if (a.n <= 4096) k_norm_backward<DT, PDT, 1, 8><<<blocks, 512, 0, s>>>(a);
        else if (a.n <= 8192) k_norm_backward<DT, PDT, 1, 16><<<blocks, 1024, 0, s>>>(a);
        else k_norm_backward<DT, PDT, 2, 16><<<blocks, 1024, 0, s>>>(a);
    }
    if (scratch)
        k_norm_params<PDT, float><<<dim3((a.n + 63) / 64, 2), 1024, 0, s>>>(a.partial, blocks, a.n, dgamma, dbeta);
    const pt_status st = check_hip(hipGetLastError(), "layerNorm gradient");
    if (scratch) scratch_free(scratch, s);
    return st;
}

}  // namespace pt

using namespace pt;

extern "C" {

pt_status pt_layernorm_backward(const void *input, const void *grad, int input_dtype, int compute_dtype, size_t rows,
                                size_t n, double eps, const void *gamma, int param_dtype, void *dinput, void *dgamma,
                                void *dbeta, pt_stream_t stream)
{
    if (!(eps > 0.0) || !isfinite(eps))
        return fail(PT_ERR_INVALID, "LayerNorm epsilon must be finite and greater than zero");
    if (compute_dtype != PT_FLOAT32 && compute_dtype != PT_FLOAT64)
        return fail(PT_ERR_INVALID, "LayerNorm compute dtype must be float32 or float64");
    if (compute_dtype == PT_FLOAT32 && (!isfinite((float)eps) || (float)eps <= 0.0f))
        return fail(PT_ERR_INVALID, "LayerNorm epsilon is not representable as float32");
    const bool half = input_dtype == PT_BFLOAT16 || input_dtype == PT_FLOAT16;
    if (compute_dtype == PT_FLOAT32 ? !half && input_dtype != PT_FLOAT32
                                    : input_dtype != PT_FLOAT64 && input_dtype != PT_FLOAT32)
        return fail(PT_ERR_INVALID, "LayerNorm gradients take float32, float16 or bfloat16 rows computed in float32, "
                                    "float64 or float32 rows computed in float64");
    if (param_dtype != compute_dtype && !(compute_dtype == PT_FLOAT32 && half && param_dtype == input_dtype))
        return fail(PT_ERR_INVALID, "LayerNorm parameters must have the compute dtype or a 16-bit input's");
    if (n == 0 && rows) return fail(PT_ERR_INVALID, "LayerNorm cannot normalize an empty dimension");
    if (n > (size_t)INT32_MAX - 16384 || rows > (size_t)INT32_MAX) return fail(PT_ERR_INVALID, "LayerNorm row too long or too many rows");
    if (rows && (!input || !grad)) return fail(PT_ERR_INVALID, "LayerNorm gradient misses an operand");
    PT_TRY(ensure_init());
    hipStream_t s = stream_of(stream);
    if (!rows) {
        // no row adds anything: the parameters' gradients are zeros
        const pt_scalar_t zero = {{0.0}, param_dtype};
        if (dgamma && n) PT_TRY(pt_fill(dgamma, param_dtype, n, &zero, stream));
        if (dbeta && n) PT_TRY(pt_fill(dbeta, param_dtype, n, &zero, stream));
        return PT_OK;
    }
    counters().fused_row_calls++;
    if (compute_dtype == PT_FLOAT64) {
        if (input_dtype == PT_FLOAT64)
            return norm_backward_general<PT_FLOAT64, PT_FLOAT64, double>(input, grad, gamma, dinput, dgamma, dbeta,
                                                                         (long long)rows, (int)n, eps, s);
        return norm_backward_general<PT_FLOAT32, PT_FLOAT64, double>(input, grad, gamma, dinput, dgamma, dbeta,
                                                                     (long long)rows, (int)n, eps, s);
    }
    const NormBwdArgs a = {input, (const float *)grad, gamma, dinput, nullptr, (long long)rows, (int)n, (float)eps};
    if (input_dtype == PT_FLOAT32) return norm_backward_f32<PT_FLOAT32, PT_FLOAT32>(a, dgamma, dbeta, s);
    const bool same = param_dtype == input_dtype;
    if (input_dtype == PT_BFLOAT16)
        return same ? norm_backward_f32<PT_BFLOAT16, PT_BFLOAT16>(a, dgamma, dbeta, s)
                    : norm_backward_f32<PT_BFLOAT16, PT_FLOAT32>(a, dgamma, dbeta, s);
    return same ? norm_backward_f32<PT_FLOAT16, PT_FLOAT16>(a, dgamma, dbeta, s)
                : norm_backward_f32<PT_FLOAT16, PT_FLOAT32>(a, dgamma, dbeta, s);
}

}  // extern "C"
