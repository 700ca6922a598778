// fp32-unit attention kernels for bf16 tensors.
#include "attn_simt.cuh"

BLOTH_INSTANTIATE_ATTN_SIMT(__nv_bfloat16)
