// Attention kernels, float16 (see pt_attention.h).
#include "../../include/pt_hip.h"

#define PT_ATTN_DT PT_FLOAT16
#include "pt_attention_inst.h"
