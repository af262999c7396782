// Backward of the norms around a block, residual streams in __bf16.
#include <hip/hip_runtime.h>

#include "include/mxmoe_block_grad.hpp"

template void mxmoe::run_block_backward<__bf16>(int, bool, const mxmoe::BlockNormArgs&, int, hipStream_t);
