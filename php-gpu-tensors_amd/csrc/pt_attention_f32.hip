// Attention kernels, float32 (see pt_attention.h).
#include "../../include/pt_hip.h"

#define PT_ATTN_DT PT_FLOAT32
#include "pt_attention_inst.h"
