// Internal declarations of the norms around a block. Not part of the public C ABI.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dmuon {

struct ResidualNorm {
  const void* x; const void* y;           // [rows][dim] of dtype; y may be NULL
  long long ld_x, ld_y;
  const void* w_pre; const void* w_post; const void* gate;   // [dim], [dim] or NULL, [groups][dim] or NULL
  int dtype, pre_dtype, post_dtype, gate_dtype;
  long long rows, rows_per_group, gates;
  int dim;
  float scale, eps;
  float2* stats;                          // [rows]: (r, s); forward: may be NULL
  void* x_new; void* h;                   // forward results; x_new may be NULL
  const void* dx_new; const void* dh;     // backward: gradients of x' and h, either may be NULL
  long long ld_dx_new, ld_dh;
  void* dx; void* dy; void* d_pre; void* d_post; void* d_gate;   // each may be NULL
  float* pre_part; float* post_part; float* gate_part;           // [blocks][dim]
  long long rows_per_block, blocks;
  int parts;                              // blocks of one gate group; 1: a block takes whole groups;
                                          // 0: no rows
  int lanes;                              // backward: rows side by side in a block
};
hipError_t launch_residual_norm(ResidualNorm a, hipStream_t stream);
// Sets rows_per_block, blocks, parts and lanes of the backward pass.
void residual_norm_split(ResidualNorm* a);
hipError_t launch_residual_norm_grad(const ResidualNorm& a, hipStream_t stream);

}  // namespace dmuon
