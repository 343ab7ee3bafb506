// self-corr-pose_amd/csrc/cross_attn_bf16.hip -- the bf16 kernels of csrc/cross_attn.hip (v_mfma_f32_32x32x16_bf16)
#include "attn_core.h"
SCP_ATTN_INSTANTIATE(__bf16)
