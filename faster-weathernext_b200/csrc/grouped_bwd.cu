// Products grouped by expert: the gradients of the pre-activation and of the weights (grouped_tile.cuh, linear_tile.cuh).
#define g_device_error g_grouped_bwd_device_error
#include "grouped_tile.cuh"

namespace fwn {

namespace {

template <int TILE, bool X32, bool SUM>
cudaError_t pre_by_act(const CUtensorMap& tb, const LinearParams& p, const GroupParams& g, int64_t items, int sms, cudaStream_t st) {
  if (p.act == 1) return launch_grouped_tile<TILE, 1, X32, false, true, SUM, kGroupRows>(tb, p, g, items, sms, st);
  if (p.act == 2) return launch_grouped_tile<TILE, 2, X32, false, true, SUM, kGroupRows>(tb, p, g, items, sms, st);
  return cudaErrorInvalidValue;  // without an activation the gradient needs no product
}
template <int TILE>
cudaError_t pre_by_type(const CUtensorMap& tb, const LinearParams& p, const GroupParams& g, int64_t items, int sms, cudaStream_t st) {
  if (p.k_blocks > p.chunk)
    return p.x_f32 ? pre_by_act<TILE, true, true>(tb, p, g, items, sms, st) : pre_by_act<TILE, false, true>(tb, p, g, items, sms, st);
  return p.x_f32 ? pre_by_act<TILE, true, false>(tb, p, g, items, sms, st) : pre_by_act<TILE, false, false>(tb, p, g, items, sms, st);
}
template <int TILE>
cudaError_t weights_by_type(const CUtensorMap& to, const LinearParams& p, const GroupParams& g, int64_t items, int sms, cudaStream_t st) {
  return p.out_f32 ? launch_grouped_tile<TILE, 0, true, true, false, false, kGroupK>(to, p, g, items, sms, st)
                   : launch_grouped_tile<TILE, 0, false, false, false, false, kGroupK>(to, p, g, items, sms, st);
}

}  // namespace

cudaError_t launch_grouped_pre_grad(int tile, const CUtensorMap& tb, const LinearParams& p, const GroupParams& g, int64_t items,
                                    int sms, cudaStream_t st) {
  if (tile == kTile256) return pre_by_type<kTile256>(tb, p, g, items, sms, st);
  if (tile == kTile256Long) return pre_by_type<kTile256Long>(tb, p, g, items, sms, st);
  if (tile == kTile128) return pre_by_type<kTile128>(tb, p, g, items, sms, st);
  return pre_by_type<kTile64>(tb, p, g, items, sms, st);
}

cudaError_t launch_grouped_weights(int tile, const CUtensorMap& to, const LinearParams& p, const GroupParams& g, int64_t items,
                                   int sms, cudaStream_t st) {
  if (tile == kTile256Long) return weights_by_type<kTile256Long>(to, p, g, items, sms, st);
  if (tile == kTile128) return weights_by_type<kTile128>(to, p, g, items, sms, st);
  return weights_by_type<kTile64>(to, p, g, items, sms, st);
}

cudaError_t take_grouped_bwd_error(unsigned int* word) {
  cudaError_t e = cudaMemcpyFromSymbol(word, g_device_error, sizeof(*word));
  if (e != cudaSuccess) return e;
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
}

}  // namespace fwn
