// Launch interface of the routing of rows to experts (routing.cu), called by routing_abi.cu.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace fwn {

constexpr int kRouteTopMax = 16;
constexpr int kRouteRows = 128;  // rows of a block

struct RouteParams {
  const void* logits;    // [rows, experts], row stride `stride`, float32 or bf16
  bool bf16_logits;
  int64_t rows, stride;
  int experts, top;
  int32_t* chosen;       // [rows, top]
  float* weights;        // [rows, top]
  int32_t* order;        // [rows top]
  int32_t* position;     // [rows, top]
  int32_t* offsets;      // [experts + 1]
  int32_t* counts;       // [experts, blocks]: workspace where rows > kRouteRows
  int32_t* totals;       // [experts]: workspace
};
inline int64_t route_blocks(int64_t rows) { return (rows + kRouteRows - 1) / kRouteRows; }
cudaError_t launch_route(const RouteParams& p, cudaStream_t stream);

// d_logits [rows, experts] (in the logits' type, contiguous) of the weights' gradient.
cudaError_t launch_route_bwd(const float* weights, const int32_t* chosen, const float* d_weights, int64_t rows, int experts,
                             int top, void* d_logits, bool bf16_logits, cudaStream_t stream);

// Rows of `d` values, float32 or bf16. `wide`, `pairs`: every row of each tensor starts where 8 (2) values are one access.
struct RowMoveParams {
  const void* x;         // [rows, d], row stride x_stride
  const void* y;         // [rows top, d] contiguous: spread's other operand of the dots, gather's rows; or null
  void* to;              // spread [rows top, d], gather [rows, d]; contiguous; or null (spread with dots alone)
  const int32_t* position;  // [rows, top]
  const float* weights;  // [rows, top] or null: ones
  float* dots;           // [rows, top] or null: x[r] . y[position[r, j]]
  int64_t rows, x_stride;
  int d, top;
  bool bf16_rows, wide, pairs;
};
// to[position[r, j]] = weights[r, j] x[r], and the dots.
cudaError_t launch_spread(const RowMoveParams& p, cudaStream_t stream);
// to[r] = sum over j of weights[r, j] y[position[r, j]].
cudaError_t launch_gather(const RowMoveParams& p, cudaStream_t stream);

cudaError_t take_routing_error(unsigned int* word);

}  // namespace fwn
