// Per-head kernel instantiations for element type __nv_bfloat16, positions of several axes.
#include "heads_inst.cuh"

BLOTH_INSTANTIATE_HEADS_AX(__nv_bfloat16, true)
