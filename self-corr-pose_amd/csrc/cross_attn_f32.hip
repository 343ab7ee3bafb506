// self-corr-pose_amd/csrc/cross_attn_f32.hip -- the fp32 kernels of csrc/cross_attn.hip (v_mfma_f32_32x32x2_f32)
#include "attn_core.h"
SCP_ATTN_INSTANTIATE(float)
