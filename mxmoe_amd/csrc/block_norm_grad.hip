// Backward of the norms around a block: entry points, and the launch that adds up the workgroups' sums (kernel: mxmoe_block_grad.hpp).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mxmoe_amd.h"
#include "include/mxmoe_block_norm.hpp"
#include "include/mxmoe_error.hpp"

namespace mxmoe {

struct ColumnSumArgs {
  const float* partial;  // [groups][planes][K]
  int groups, planes, K, wtype;
  float factor;
  const void* scale;
  const void* w1;
  void* grad_w2;         // from plane 0
  void* grad_w1;         // from plane 1
  void* grad_scale;
};
// 32 columns a workgroup (128 bytes of every partial row), 32 threads a column: sixteen rows each of 512, in two rounds of loads.
__global__ void __launch_bounds__(1024) column_sum_kernel(const ColumnSumArgs a) {
  __shared__ float part[32][33];
  const int col = threadIdx.x & 31, sub = threadIdx.x >> 5, plane = blockIdx.y;
  if (plane == 0 ? !a.grad_w2 : !a.grad_w1 && !a.grad_scale) return;
  const int c = blockIdx.x * 32 + col;
  float s = 0.0f;
  if (c < a.K) {
    const float* p = a.partial + (long)plane * a.K + c;
    const long ld = (long)a.planes * a.K;
#pragma unroll 8
    for (int g = sub; g < a.groups; g += 32) s += p[g * ld];
  }
  part[sub][col] = s;
  __syncthreads();
  if (sub || c >= a.K) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) s += part[i][col];
  if (plane == 0) {
    store_of(a.wtype, a.grad_w2, c, s);
  } else {
    if (a.grad_w1) store_of(a.wtype, a.grad_w1, c, s * (a.scale ? a.factor * load_of(a.wtype, a.scale, c) : a.factor));
    if (a.grad_scale) store_of(a.wtype, a.grad_scale, c, s * (a.w1 ? a.factor * load_of(a.wtype, a.w1, c) : a.factor));
  }
}

static int run_backward(int xtype, int ztype, bool has_z, BlockNormArgs& a, void* grad_w2, void* grad_w1, void* grad_scale, hipStream_t s) {
  a.grad_w2 = grad_w2;
  a.grad_w1 = grad_w1;
  a.grad_scale = grad_scale;
  const int grid = backward_groups(a.T, a.K);
  if (grid > 0) {
    if (xtype == kF16) run_block_backward<_Float16>(ztype, has_z, a, grid, s);
    else if (xtype == kF32) run_block_backward<float>(ztype, has_z, a, grid, s);
    else run_block_backward<__bf16>(ztype, has_z, a, grid, s);
  }
  if (grid != 1 && (grad_w2 || grad_w1 || grad_scale)) {  // (no tokens: the sums are zero, and are written)
    const int planes = has_z ? 2 : 1;
    const ColumnSumArgs c{a.partial, grid, planes, a.K, a.wtype, a.factor, a.scale, a.w1, grad_w2, grad_w1, grad_scale};
    hipLaunchKernelGGL(column_sum_kernel, dim3((a.K + 31) / 32, planes), dim3(1024), 0, s, c);
  }
  return launched();
}
static int null_pointer() { return refuse(5, "null pointer"); }

}  // namespace mxmoe

using namespace mxmoe;

extern "C" {

size_t mxmoe_block_backward_workspace_bytes(int num_tokens, int K) {
  if (num_tokens <= 0 || K < 1 || K > kMaxNormRow) return 0;
  const int groups = backward_groups(num_tokens, K);
  return groups > 1 ? (size_t)groups * 2 * (size_t)K * sizeof(float) : 0;
}

int mxmoe_block_norm_backward(const void* grad_y, int64_t ld_grad_y, int y_dtype, const void* x, int64_t ldx, int x_dtype, const void* weight, int weight_dtype, const void* grad_residual,
                              int64_t ld_grad_residual, float eps, int num_tokens, int K, void* grad_x, void* grad_weight, void* workspace, void* stream) {
  BlockNormArgs a{};
  a.x = x;
  a.ldx = (long)ldx;
  a.grad_y = grad_y;
  a.ldgy = (long)ld_grad_y;
  a.grad_h = grad_residual;
  a.ldgh = (long)ld_grad_residual;
  a.w2 = weight;
  a.wtype = weight_dtype;
  a.eps = eps;
  a.factor = 1.0f;
  a.T = num_tokens;
  a.K = K;
  a.grad_x = grad_x;
  a.partial = reinterpret_cast<float*>(workspace);
  if (const int rc = check_block_norm(a, x_dtype, y_dtype)) return rc;
  if ((weight && !grad_weight) || (num_tokens && (!grad_y || !x || !grad_x || (weight && !workspace && mxmoe_block_backward_workspace_bytes(num_tokens, K))))) return null_pointer();
  return run_backward(x_dtype, y_dtype, false, a, weight ? grad_weight : nullptr, nullptr, nullptr, (hipStream_t)stream);
}

int mxmoe_block_residual_backward(const void* grad_h, int64_t ld_grad_h, const void* grad_y, int64_t ld_grad_y, const void* x, int64_t ldx, int x_dtype, const void* z, int64_t ldz,
                                  int z_dtype, int gate_kind, const void* gate, int64_t ld_gate, int gate_dtype, int sigmoid, float factor, const void* scale, const void* norm_weight,
                                  const void* next_weight, int weight_dtype, float eps, int num_tokens, int K, void* grad_x, void* grad_z, void* grad_gate, void* grad_scale,
                                  void* grad_norm_weight, void* grad_next_weight, void* workspace, void* stream) {
  BlockNormArgs a{};
  a.x = x;
  a.z = z;
  a.gate = gate;
  a.scale = scale;
  a.w1 = norm_weight;
  a.w2 = next_weight;
  a.ldx = (long)ldx;
  a.ldz = (long)ldz;
  a.ldg = (long)ld_gate;
  a.T = num_tokens;
  a.K = K;
  a.wtype = weight_dtype;
  a.gate_kind = gate_kind;
  a.gate_type = gate_dtype;
  a.sigmoid = sigmoid != 0;
  a.eps = eps;
  a.factor = factor;
  a.grad_h = grad_h;
  a.grad_y = grad_y;
  a.ldgh = (long)ld_grad_h;
  a.ldgy = (long)ld_grad_y;
  a.grad_x = grad_x;
  a.grad_z = grad_z;
  a.grad_gate = grad_gate;
  a.partial = reinterpret_cast<float*>(workspace);
  if (const int rc = check_block_norm(a, x_dtype, z_dtype)) return rc;
  if (gate_kind == kElementGate && gate_dtype != z_dtype) return refuse(3, "a gate per element has the block output's type");
  if ((scale && !grad_scale) || (norm_weight && !grad_norm_weight) || (next_weight && !grad_next_weight)) return null_pointer();
  if (num_tokens && (!x || !z || !grad_x || !grad_z || (gate_kind && !grad_gate) || ((scale || norm_weight || next_weight) && !workspace && mxmoe_block_backward_workspace_bytes(num_tokens, K)))) return null_pointer();
  if (num_tokens && !grad_h && !grad_y) return refuse(5, "neither the gradient of h nor that of y is given");
  return run_backward(x_dtype, z_dtype, true, a, next_weight ? grad_next_weight : nullptr, norm_weight ? grad_norm_weight : nullptr, scale ? grad_scale : nullptr, (hipStream_t)stream);
}

}  // extern "C"
