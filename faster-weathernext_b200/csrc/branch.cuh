// Launch interface of the branch kernels (branch.cu, branch_bwd_f32.cu, branch_bwd_bf16.cu), called by branch_abi.cu.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "philox.cuh"
#include "rms.cuh"

namespace fwn {

constexpr int kBranchMaxWidth = 8192;  // rows of widths off 8: 7 less

struct BranchParams {
  const void* x;            // [rows, d], row stride x_stride
  const void* y;            // [rows, d], row stride y_stride
  const void* post_weight;  // [d] or null
  const void* weight;       // [d] or null
  const void* gate;         // [rows / gate_span, d] or null
  void* s;                  // [rows, d] in x's type
  void* h;                  // [rows, d]
  float* scale;             // [rows], e4m3 output only
  float* rstd;              // [rows, 2]: of y and of s; or null
  int64_t rows, x_stride, y_stride, gate_span;
  int d;
  float eps, alpha;
  int out_type;             // RmsOut
  bool x_bf16, y_bf16, post_bf16, weight_bf16, gate_bf16;
  bool wide;                // rows of whole wide accesses; else contiguous rows of any width
  int sms;
  DropParams drop;
};

struct BranchBwdParams {
  const void *x, *y, *post_weight, *weight, *gate;
  const float* rstd;
  const void* dh;           // [rows, d] or null
  const void* ds;           // [rows, d] in x's type or null
  void* dx;                 // outputs: each may be null
  void* dy;
  void* d_post;
  void* d_weight;
  void* d_gate;
  float* part_u;            // [gates * slices, d]: with d_gate (of fewer rows than x) or d_post
  float* part_w;            // [blocks, d]: with d_weight
  int64_t rows, x_stride, y_stride, gate_span;
  int d;
  float alpha;
  bool x_bf16, y_bf16, post_bf16, weight_bf16, gate_bf16, dh_bf16;
  bool wide, gate_values;   // gate_values: a gate of its own for every row
  int gates, slices, blocks;
  DropParams drop;
};

cudaError_t launch_branch(const BranchParams& p, cudaStream_t stream);

// Blocks, and slices of each gate's rows, of the gradient's kernel.
void branch_bwd_shape(int64_t rows, int d, int gates, int sms, bool wide, int* slices, int* blocks);
cudaError_t launch_branch_bwd_f32(const BranchBwdParams& p, cudaStream_t stream);   // a float32 stream
cudaError_t launch_branch_bwd_bf16(const BranchBwdParams& p, cudaStream_t stream);  // a bf16 one
cudaError_t launch_branch_bwd_finish(const BranchBwdParams& p, cudaStream_t stream);

// out[i] = x[i] under the mask, i < n; x, out bf16 or float32, `wide`: both start where 8 values are one access.
cudaError_t launch_dropout(const void* x, void* out, int64_t n, bool bf16_values, bool wide, const DropParams& drop,
                           cudaStream_t stream);

}  // namespace fwn
