// Instances of the attention kernels of one element type PT_ATTN_DT and
// their launches (included by pt_attention_{bf16,f16,f32}.hip, one unit per
// type so that they build side by side).
#include "pt_attention.h"

namespace pt {

template <int DP, int RW, bool VEC>
static void launch_fwd(const AttnArgs &g, unsigned blocks, hipStream_t s)
{
    if constexpr (AttnFwdShape<PT_ATTN_DT, DP, RW>::kBuilt)
        k_attention<PT_ATTN_DT, DP, RW, VEC><<<dim3(blocks, (unsigned)g.splits), 256, 0, s>>>(g);
}

template <int DP, bool VEC>
static void launch_dkv(const AttnArgs &g, unsigned blocks, hipStream_t s)
{
    if constexpr (AttnBwdShape<PT_ATTN_DT, DP>::kSplitPasses) {
        k_attention_dkv<PT_ATTN_DT, DP, 1, VEC><<<blocks, 256, 0, s>>>(g);
        k_attention_dkv<PT_ATTN_DT, DP, 2, VEC><<<blocks, 256, 0, s>>>(g);
    } else {
        k_attention_dkv<PT_ATTN_DT, DP, 0, VEC><<<blocks, 256, 0, s>>>(g);
    }
}

template <int DP, bool VEC>
static void launch_dq(const AttnArgs &g, unsigned blocks, hipStream_t s)
{
    k_attention_dq<PT_ATTN_DT, DP, VEC><<<blocks, 256, 0, s>>>(g);
}

// F<DP, VEC>: the smallest built head size that holds g.size
#define PT_ATTN_BY_SIZE(F, ...)                                        \
    do {                                                               \
        if (g.size <= 64) vec ? F<64 __VA_ARGS__, true>(g, blocks, s) : F<64 __VA_ARGS__, false>(g, blocks, s);     \
        else if (g.size <= 128) vec ? F<128 __VA_ARGS__, true>(g, blocks, s) : F<128 __VA_ARGS__, false>(g, blocks, s); \
        else vec ? F<256 __VA_ARGS__, true>(g, blocks, s) : F<256 __VA_ARGS__, false>(g, blocks, s);                \
    } while (0)
#define PT_COMMA ,

template <> bool attention_narrow_built<PT_ATTN_DT>(int size)
{
    return size <= 64    ? AttnFwdShape<PT_ATTN_DT, 64, 1>::kBuilt
           : size <= 128 ? AttnFwdShape<PT_ATTN_DT, 128, 1>::kBuilt
                         : AttnFwdShape<PT_ATTN_DT, 256, 1>::kBuilt;
}

template <> void launch_attention<PT_ATTN_DT>(const AttnArgs &g, bool narrow, bool vec, unsigned blocks, hipStream_t s)
{
    if (narrow) PT_ATTN_BY_SIZE(launch_fwd, PT_COMMA 1);
    else PT_ATTN_BY_SIZE(launch_fwd, PT_COMMA 4);
}

template <> void launch_attention_dkv<PT_ATTN_DT>(const AttnArgs &g, bool vec, unsigned blocks, hipStream_t s)
{
    PT_ATTN_BY_SIZE(launch_dkv, );
}

template <> void launch_attention_dq<PT_ATTN_DT>(const AttnArgs &g, bool vec, unsigned blocks, hipStream_t s)
{
    PT_ATTN_BY_SIZE(launch_dq, );
}

}  // namespace pt
