// Backward of the norms around a block, residual streams in float.
#include <hip/hip_runtime.h>

#include "include/mxmoe_block_grad.hpp"

template void mxmoe::run_block_backward<float>(int, bool, const mxmoe::BlockNormArgs&, int, hipStream_t);
