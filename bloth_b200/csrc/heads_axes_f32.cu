// Per-head kernel instantiations for element type float, positions of several axes.
#include "heads_inst.cuh"

BLOTH_INSTANTIATE_HEADS_AX(float, true)
