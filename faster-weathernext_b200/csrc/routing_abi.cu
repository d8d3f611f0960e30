// C ABI of the routing of rows to experts (include/fwn_attn.h): argument checks and launches.
#include <algorithm>

#include "abi.cuh"
#include "grouped.cuh"
#include "routing.cuh"

using namespace fwn;

namespace {

fwn_status check_route(const fwn_route_desc* d) {
  if (!d) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "desc is null");
  if (d->rows < 0 || d->experts <= 0 || d->top <= 0 || d->top > d->experts)
    return abi_fail(FWN_ERR_INVALID_ARGUMENT, "bad rows=%lld, experts=%d or top=%d", static_cast<long long>(d->rows), d->experts, d->top);
  if (d->experts > kGroupsMax || d->top > kRouteTopMax)
    return abi_fail(FWN_ERR_UNSUPPORTED, "experts=%d or top=%d exceeds %d or %d", d->experts, d->top, kGroupsMax, kRouteTopMax);
  if (d->rows * d->top > INT32_MAX) return abi_fail(FWN_ERR_UNSUPPORTED, "rows=%lld too large", static_cast<long long>(d->rows));
  if (!abi_float(d->dtype)) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "logits and rows are bf16 or float32 (got dtype %d)", d->dtype);
  return FWN_OK;
}

fwn_status check_move(const fwn_route_desc* d, int32_t width, int64_t x_stride, bool strided) {
  if (fwn_status s = check_route(d); s != FWN_OK) return s;
  if (width <= 0) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "bad d=%d", width);
  if (strided && d->rows > 1 && x_stride < width) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "the row stride is below d");
  return FWN_OK;
}

RowMoveParams move_of(const fwn_route_desc& d, int32_t width, const int32_t* position, const float* weights) {
  RowMoveParams p{};
  p.position = position;
  p.weights = weights;
  p.rows = d.rows;
  p.d = width;
  p.top = d.top;
  p.bf16_rows = d.dtype == FWN_DTYPE_BF16;
  return p;
}
// Whether rows of `width` values, `stride` apart, of these tensors start where n values are one access.
bool rows_start(int n, int32_t dtype, int32_t width, int64_t stride, std::initializer_list<const void*> tensors) {
  if (width % n != 0 || stride % n != 0) return false;
  for (const void* t : tensors)
    if (!abi_aligned(t, n * abi_size(dtype))) return false;
  return true;
}

}  // namespace

extern "C" {

fwn_status fwn_route_workspace_size(const fwn_route_desc* desc, size_t* bytes) {
  if (!bytes) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "bytes is null");
  if (fwn_status s = check_route(desc); s != FWN_OK) return s;
  const int64_t blocks = route_blocks(desc->rows);
  *bytes = blocks > 1 ? static_cast<size_t>(blocks + 1) * desc->experts * sizeof(int32_t) : 0;
  return abi_ok();
}

fwn_status fwn_route(const fwn_route_desc* desc, const void* logits, int64_t stride, int32_t* experts, float* weights,
                     int32_t* order, int32_t* position, int32_t* offsets, void* workspace, size_t workspace_bytes, void* stream) {
  fwn_status s = check_route(desc);
  if (s != FWN_OK) return s;
  const fwn_route_desc& d = *desc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!offsets) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "null pointer");
  if ((s = abi_elements({{logits, abi_size(d.dtype)}, {experts, 4}, {weights, 4}, {order, 4}, {position, 4}, {offsets, 4}, {workspace, 4}})) != FWN_OK)
    return s;
  if (d.rows == 0) {
    cudaError_t e = cudaMemsetAsync(offsets, 0, (d.experts + 1) * sizeof(int32_t), st);
    if (e != cudaSuccess) return abi_cuda_fail(e, "clear offsets");
    return abi_ok();
  }
  if (!logits || !experts || !weights || !order || !position) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "null pointer");
  if (d.rows > 1 && stride < d.experts) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "the row stride is below the number of experts");
  size_t need = 0;
  if ((s = fwn_route_workspace_size(desc, &need)) != FWN_OK) return s;
  if (need > 0 && (!workspace || workspace_bytes < need)) return abi_fail(FWN_ERR_WORKSPACE, "workspace of %zu bytes needed", need);
  RouteParams p{};
  p.logits = logits;
  p.bf16_logits = d.dtype == FWN_DTYPE_BF16;
  p.rows = d.rows;
  p.stride = stride;
  p.experts = d.experts;
  p.top = d.top;
  p.chosen = experts;
  p.weights = weights;
  p.order = order;
  p.position = position;
  p.offsets = offsets;
  p.counts = static_cast<int32_t*>(workspace);
  p.totals = need > 0 ? p.counts + route_blocks(d.rows) * d.experts : nullptr;
  cudaError_t e = launch_route(p, st);
  if (e != cudaSuccess) return abi_cuda_fail(e, "route");
  return abi_ok();
}

fwn_status fwn_route_bwd(const fwn_route_desc* desc, const float* weights, const int32_t* experts, const float* d_weights,
                         void* d_logits, void* stream) {
  if (fwn_status s = check_route(desc); s != FWN_OK) return s;
  const fwn_route_desc& d = *desc;
  if (d.rows == 0) return abi_ok();
  if (!weights || !experts || !d_weights || !d_logits) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "null pointer");
  if (fwn_status s = abi_elements({{weights, 4}, {experts, 4}, {d_weights, 4}, {d_logits, abi_size(d.dtype)}}); s != FWN_OK) return s;
  cudaError_t e = launch_route_bwd(weights, experts, d_weights, d.rows, d.experts, d.top, d_logits, d.dtype == FWN_DTYPE_BF16,
                                   static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return abi_cuda_fail(e, "route_bwd");
  return abi_ok();
}

fwn_status fwn_route_spread(const fwn_route_desc* desc, int32_t width, const void* x, int64_t x_stride, const int32_t* position,
                            const float* weights, const void* y, void* out, float* dots, void* stream) {
  if (fwn_status s = check_move(desc, width, x_stride, true); s != FWN_OK) return s;
  const fwn_route_desc& d = *desc;
  if ((y != nullptr) != (dots != nullptr)) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "y and dots come together");
  if (d.rows == 0) return abi_ok();
  if (!x || !position || (!out && !dots)) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "null pointer");
  const int64_t es = abi_size(d.dtype);
  if (fwn_status s = abi_elements({{x, es}, {y, es}, {out, es}, {position, 4}, {weights, 4}, {dots, 4}}); s != FWN_OK) return s;
  RowMoveParams p = move_of(d, width, position, weights);
  p.x = x;
  p.x_stride = x_stride;
  p.y = y;
  p.to = out;
  p.dots = dots;
  const int64_t stride = d.rows == 1 ? width : x_stride;
  p.wide = rows_start(8, d.dtype, width, stride, {x, y, out});
  p.pairs = rows_start(2, d.dtype, width, stride, {x, y, out});
  cudaError_t e = launch_spread(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return abi_cuda_fail(e, "route_spread");
  return abi_ok();
}

fwn_status fwn_route_gather(const fwn_route_desc* desc, int32_t width, const void* y, const int32_t* position, const float* weights,
                            void* out, void* stream) {
  if (fwn_status s = check_move(desc, width, 0, false); s != FWN_OK) return s;
  const fwn_route_desc& d = *desc;
  if (d.rows == 0) return abi_ok();
  if (!y || !position || !out) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "null pointer");
  const int64_t es = abi_size(d.dtype);
  if (fwn_status s = abi_elements({{y, es}, {out, es}, {position, 4}, {weights, 4}}); s != FWN_OK) return s;
  RowMoveParams p = move_of(d, width, position, weights);
  p.y = y;
  p.to = out;
  p.wide = rows_start(8, d.dtype, width, width, {y, out});
  p.pairs = rows_start(2, d.dtype, width, width, {y, out});
  cudaError_t e = launch_gather(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return abi_cuda_fail(e, "route_gather");
  return abi_ok();
}

}  // extern "C"
