// Instances of the attention kernels of one element type PT_ATTN_DT and
// their launches (included by pt_attention_{bf16,f16,f32}.hip, one unit per
// type so that they build side by side).
#include "pt_attention.h"

namespace pt {

template <int DP, bool VEC>
static void launch_fwd(const AttnArgs &g, unsigned blocks, hipStream_t s)
{
    k_attention<PT_ATTN_DT, DP, VEC><<<dim3(blocks, (unsigned)g.splits), 256, 0, s>>>(g);
}

template <int DP>
static void launch_token(const AttnArgs &g, unsigned blocks, hipStream_t s)
{
    k_attention_token<PT_ATTN_DT, DP><<<dim3(blocks, (unsigned)g.splits), 64 * AttnTokenShape<PT_ATTN_DT, DP>::NW, 0, s>>>(g);
}

template <int DP, bool VEC>
static void launch_dkv(const AttnArgs &g, unsigned blocks, hipStream_t s)
{
    if constexpr (AttnBwdShape<PT_ATTN_DT, DP>::kSplitPasses) {
        k_attention_dkv<PT_ATTN_DT, DP, 1, VEC><<<dim3(blocks, (unsigned)g.splits), 256, 0, s>>>(g);
        k_attention_dkv<PT_ATTN_DT, DP, 2, VEC><<<dim3(blocks, (unsigned)g.splits), 256, 0, s>>>(g);
    } else {
        k_attention_dkv<PT_ATTN_DT, DP, 0, VEC><<<dim3(blocks, (unsigned)g.splits), 256, 0, s>>>(g);
    }
}

template <int DP, bool VEC>
static void launch_dq(const AttnArgs &g, unsigned blocks, hipStream_t s)
{
    k_attention_dq<PT_ATTN_DT, DP, VEC><<<dim3(blocks, (unsigned)g.splits), 256, 0, s>>>(g);
}

// F<DP, VEC>: the smallest built head size that holds g.size
#define PT_ATTN_BY_SIZE(F)                                                     \
    do {                                                                       \
        if (g.size <= 64) vec ? F<64, true>(g, blocks, s) : F<64, false>(g, blocks, s);        \
        else if (g.size <= 128) vec ? F<128, true>(g, blocks, s) : F<128, false>(g, blocks, s); \
        else vec ? F<256, true>(g, blocks, s) : F<256, false>(g, blocks, s);   \
    } while (0)

template <> int attention_backward_tile<PT_ATTN_DT>(int size)
{
    return size <= 64    ? AttnBwdShape<PT_ATTN_DT, 64>::BN
           : size <= 128 ? AttnBwdShape<PT_ATTN_DT, 128>::BN
                         : AttnBwdShape<PT_ATTN_DT, 256>::BN;
}

template <> void launch_attention<PT_ATTN_DT>(const AttnArgs &g, bool token, bool vec, unsigned blocks, hipStream_t s)
{
    if (!token) PT_ATTN_BY_SIZE(launch_fwd);
    else if (g.size <= 64) launch_token<64>(g, blocks, s);
    else if (g.size <= 128) launch_token<128>(g, blocks, s);
    else launch_token<256>(g, blocks, s);
}

template <> void launch_attention_dkv<PT_ATTN_DT>(const AttnArgs &g, bool vec, unsigned blocks, hipStream_t s)
{
    PT_ATTN_BY_SIZE(launch_dkv);
}

template <> void launch_attention_dq<PT_ATTN_DT>(const AttnArgs &g, bool vec, unsigned blocks, hipStream_t s)
{
    PT_ATTN_BY_SIZE(launch_dq);
}

}  // namespace pt
