// Products grouped by expert: the forward, and the gradient of the rows (grouped_tile.cuh, linear_tile.cuh).
#define g_device_error g_grouped_fwd_device_error
#include "grouped_tile.cuh"

namespace fwn {

namespace {

template <int TILE, bool O32, bool SUM>
cudaError_t by_act(const CUtensorMap& tb, const LinearParams& p, const GroupParams& g, int64_t items, int sms, cudaStream_t st) {
  if (p.act == 1) return launch_grouped_tile<TILE, 1, O32, O32, false, SUM, kGroupRows>(tb, p, g, items, sms, st);
  if (p.act == 2) return launch_grouped_tile<TILE, 2, O32, O32, false, SUM, kGroupRows>(tb, p, g, items, sms, st);
  return launch_grouped_tile<TILE, 0, O32, O32, false, SUM, kGroupRows>(tb, p, g, items, sms, st);
}
template <int TILE>
cudaError_t by_type(const CUtensorMap& tb, const LinearParams& p, const GroupParams& g, int64_t items, int sms, cudaStream_t st) {
  if (!p.out_f32) return by_act<TILE, false, false>(tb, p, g, items, sms, st);
  return p.k_blocks > p.chunk ? by_act<TILE, true, true>(tb, p, g, items, sms, st) : by_act<TILE, true, false>(tb, p, g, items, sms, st);
}

}  // namespace

cudaError_t launch_grouped_forward(int tile, const CUtensorMap& tb, const LinearParams& p, const GroupParams& g, int64_t items,
                                   int sms, cudaStream_t st) {
  if (tile == kTile256) return by_type<kTile256>(tb, p, g, items, sms, st);
  if (tile == kTile256Long) return by_type<kTile256Long>(tb, p, g, items, sms, st);
  if (tile == kTile128) return by_type<kTile128>(tb, p, g, items, sms, st);
  return by_type<kTile64>(tb, p, g, items, sms, st);
}

cudaError_t take_grouped_fwd_error(unsigned int* word) {
  cudaError_t e = cudaMemcpyFromSymbol(word, g_device_error, sizeof(*word));
  if (e != cudaSuccess) return e;
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
}

}  // namespace fwn
