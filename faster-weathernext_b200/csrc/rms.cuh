// Launch interface of the RMS norm kernels (rms.cu), called by the C ABI (fwn_attn.cu).
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace fwn {

enum RmsOut { kRmsBf16 = 0, kRmsF32 = 1, kRmsE4m3 = 2 };

constexpr int kRmsMaxWidth = 16384;

struct RmsParams {
  const void* x;         // [rows, d], row stride x_stride (elements)
  const void* residual;  // [rows, d], row stride residual_stride; or null
  const void* weight;    // [d] or null
  void* x_out;           // [rows, d] in x's type, with a residual only
  void* out;             // [rows, d]
  float* scale;          // [rows], e4m3 output only
  int64_t rows, x_stride, residual_stride;
  int d;
  float eps;
  int out_type;
  bool x_bf16, residual_bf16, weight_bf16;
  bool normalize;        // false: the sum itself (scaled by weight, if any) is written
  int mode, sms;         // rms_mode; multiprocessors
};

struct RmsBwdParams {
  const void* x;         // what was normalised, or x of it when `residual` is given (then x + residual was)
  const void* residual;
  const void* weight;
  const void* dh;        // [rows, d]
  const void* ds;        // [rows, d] in x's type: gradient of the stored sum, or null
  void* dx;              // [rows, d] in x's type, or null
  void* dr;              // [rows, d] in the residual's type, or null
  float* part;           // [blocks, d] with dw, else null
  void* dw;              // [d]
  int64_t rows, x_stride, residual_stride;
  int d;
  float eps;
  bool x_bf16, residual_bf16, weight_bf16, dh_bf16, dw_bf16;
  int mode;
};

// How rows are laid over threads. wide: every row of every tensor allows 8 values per access; packed: all tensors are
// contiguous, from a base that allows 8 values per access.
int rms_mode(bool wide, bool packed, int d);
cudaError_t launch_rms_norm(const RmsParams& p, cudaStream_t stream);
int rms_bwd_blocks(int64_t rows, int d, int sms, int mode, bool x_bf16);
cudaError_t launch_rms_norm_bwd(const RmsBwdParams& p, int blocks, cudaStream_t stream);
cudaError_t launch_column_sum(const float* part, int64_t rows, int d, void* out, bool out_bf16, cudaStream_t stream);

}  // namespace fwn
