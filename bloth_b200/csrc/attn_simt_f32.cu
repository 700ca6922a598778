// fp32-unit attention kernels for f32 tensors.
#include "attn_simt.cuh"

BLOTH_INSTANTIATE_ATTN_SIMT(float)
