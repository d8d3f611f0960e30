// The tensor-core kernel over products grouped by expert (linear_tile.cuh's body, walked by GroupWalk), and its launch.
//
// Bound and tiles as the plain product's (linear_tile.cuh). Measured at 81,924 x 512 x 2,048 over 1 / 8 / 64 experts (plain):
// GELU 152 / 154 / 169 us (146), act'() with column sums 228 / 232 / 240 (224), d_a 120 / 123 / 134 (120), the weights' gradient
// 124 / 136 / 137 (124), of uneven experts 132 over 8 and 163 over 64, and its parts' sum 4 / 17 / 0.
#pragma once

#include "grouped.cuh"
#include "linear_tile.cuh"

namespace fwn {

namespace {

// tm: the map that is not an expert's, b's (kGroupRows) or out's (kGroupK).
template <int TILE, int ACT, bool X32, bool O32, bool PRE, bool SUM, int GROUP>
__global__ void __launch_bounds__(LinearCfg<TILE, X32, O32, PRE, SUM>::THREADS, 1)
    grouped_tile_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ LinearParams p,
                        const __grid_constant__ GroupParams gp) {
  linear_tile_body<TILE, ACT, X32, O32, PRE, SUM, GROUP>(tm, tm, tm, tm, p, gp);
}

// `items`: at most so many tiles (their number is known on the device alone).
template <int TILE, int ACT, bool X32, bool O32, bool PRE, bool SUM, int GROUP>
cudaError_t launch_grouped_tile(const CUtensorMap& tm, const LinearParams& given, const GroupParams& gp, int64_t items, int sms,
                                cudaStream_t stream) {
  LinearParams p = given;
  using C = LinearCfg<TILE, X32, O32, PRE, SUM>;
  auto kernel = grouped_tile_kernel<TILE, ACT, X32, O32, PRE, SUM, GROUP>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  const int groups = static_cast<int>(std::min<int64_t>(items, sms / C::CG));
  p.step_n = groups % p.n_tiles;
  p.step_m = groups / p.n_tiles;
  p.step_s = 0;
  if (GROUP == kGroupK) {
    p.step_s = p.step_m / p.m_tiles;
    p.step_m %= p.m_tiles;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(groups * C::CG);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C::CG;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, tm, p, gp);
}

}  // namespace

}  // namespace fwn
