// Per-head kernel instantiations for element type __half, positions of several axes.
#include "heads_inst.cuh"

BLOTH_INSTANTIATE_HEADS_AX(__half, true)
