// Launch interface of the projection kernels (linear.cu), called by the C ABI (fwn_attn.cu).
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

namespace fwn {

// Shapes of the tensor-core kernel's output tile: two SMs on 256 x 256 (two forms: sixteen epilogue warps and four
// stages, or eight and five), one on 128 x 128 or 128 x 64.
enum LinearTile { kTile256 = 0, kTile256Long = 1, kTile128 = 2, kTile64 = 3, kLinearTiles = 4 };
__host__ __device__ constexpr bool linear_pair(int t) { return t == kTile256 || t == kTile256Long; }
__host__ __device__ constexpr int linear_tile_m(int t) { return linear_pair(t) ? 256 : 128; }
__host__ __device__ constexpr int linear_tile_n(int t) { return linear_pair(t) ? 256 : t == kTile128 ? 128 : 64; }
// Columns of the output (and of x) that an epilogue warp takes at a time: 128 bytes of a row where the warp's half of
// the tile has them; the boxes of the two tensor maps.
__host__ __device__ constexpr int linear_chunk_cols(int t, bool f32) { return f32 || t == kTile64 ? 32 : 64; }
// Rows of B that one CTA loads (and the box rows of its tensor map).
__host__ __device__ constexpr int linear_box_n(int t) { return linear_tile_n(t) / (linear_pair(t) ? 2 : 1); }
// Stages of k (128 bytes each: 64 bf16) that a float32 result accumulates in the tensor core at a time (linear.cu).
constexpr int kLinearChunk = 12;

struct LinearParams {
  const void* bias;      // [n] or null
  const float* a_scale;  // [m] / [n]: 8-bit operands; else null
  const float* b_scale;
  const void* x;         // residual, or the gradient of the output (pre_grad); [m, n], row stride ldx; or null
  void* out;             // [m, n], row stride ldo
  float* colsum;         // pre_grad: [ceil(m / 32), n] sums of 32 rows each; or null
  int64_t m, ldx, ldo;
  int n, k;
  int act;               // 0 none, 1 GELU (tanh form), 2 swish
  bool bias_bf16, x_f32, out_f32;
  bool pre_grad;         // out = x act'(a b + bias) in bf16 instead of act(a b + bias) + x
  bool fp8;              // e4m3 operands (bf16 otherwise)
  bool a_mn, b_mn;       // the operand's m (n) is contiguous instead of its k
  bool x_direct, out_direct;  // rows that TMA cannot address (strides or base off 16 bytes): plain accesses
  int m_tiles, n_tiles, splits, k_blocks, items;
  int chunk;             // stages of k per accumulation in the tensor core (float32 output)
  // Set at the launch: the stages of k of a split (the first kb_r take one more), and the walk's step in tiles.
  int kb_q, kb_r, step_n, step_m, step_s;
  int64_t split_rows;    // rows of one split's partial sums in the output (splits > 1)
};

cudaError_t launch_linear_tiles(int tile, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tx,
                                const CUtensorMap& to, const LinearParams& p, int sms, cudaStream_t stream);
// out = epilogue(sum over splits of part); p as of the whole product, part [splits, split_rows, ldp].
cudaError_t launch_linear_split_sum(const float* part, int64_t ldp, const LinearParams& p, cudaStream_t stream);

constexpr int kLinearRowsMax = 8;
// m <= kLinearRowsMax rows, both operands with k contiguous.
cudaError_t launch_linear_rows(const void* a, int64_t lda, const void* b, int64_t ldb, bool wide, const LinearParams& p,
                               cudaStream_t stream);

// dst[r, 0..cols) = src[r, 0..cols) for elements of `es` (1 or 2) bytes; dst 16-byte aligned, its rows ldd apart, a multiple
// of 16 bytes.
cudaError_t launch_pack_rows(const void* src, int64_t lds, void* dst, int64_t ldd, int64_t rows, int64_t cols, int es,
                             cudaStream_t stream);

// Column sums of x [m, n] (bf16 or float32) into part [blocks, n], and (cast not null) x rounded to bf16.
int grad_cast_blocks(int64_t m, int n, int sms);
cudaError_t launch_grad_cast(const void* x, bool x_f32, int64_t ldx, int64_t m, int n, void* cast, int64_t ldc,
                             float* part, int blocks, bool wide, cudaStream_t stream);

// The device error word of linear.cu's kernels (read and cleared, after the stream was synchronised).
cudaError_t take_linear_error(unsigned int* word);

}  // namespace fwn
