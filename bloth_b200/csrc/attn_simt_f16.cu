// fp32-unit attention kernels for f16 tensors.
#include "attn_simt.cuh"

BLOTH_INSTANTIATE_ATTN_SIMT(__half)
