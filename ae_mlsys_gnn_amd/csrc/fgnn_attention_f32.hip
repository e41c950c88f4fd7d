// The attention kernels of one element type.
#include "fgnn_attention.h"
template void at_launch<float>(int what, const AtShape &shape, const AttentionP &p, unsigned grid, hipStream_t st);
