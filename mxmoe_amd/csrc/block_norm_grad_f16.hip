// Backward of the norms around a block, residual streams in _Float16.
#include <hip/hip_runtime.h>

#include "include/mxmoe_block_grad.hpp"

template void mxmoe::run_block_backward<_Float16>(int, bool, const mxmoe::BlockNormArgs&, int, hipStream_t);
