// Projections: out = act(a b^T + bias) + residual over any m, n, k, bf16 or 8-bit operands, and what their gradients
// need.
//
// linear_tile_kernel, the tensor-core kernel (tcgen05, TMA, TMEM), takes every product of more than kLinearRowsMax
// rows: the forward, d_a = d_pre b, d_b = d_pre^T a (an operand's k or its m / n may be the contiguous dimension: both
// orders of the shared-memory descriptors), and d_pre = dy act'(a b^T + bias) with its column sums, which recomputes
// the pre-activation instead of keeping it. linear_rows_kernel takes the few rows of a serving call.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

// This translation unit's device error word.
#define g_device_error g_linear_device_error
#include "linear_tile.cuh"

namespace fwn {

namespace {

template <int TILE, int ACT, bool X32, bool O32, bool PRE, bool SUM>
__global__ void __launch_bounds__(LinearCfg<TILE, X32, O32, PRE, SUM>::THREADS, 1)
    linear_tile_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                       const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_o,
                       const __grid_constant__ LinearParams p) {
  linear_tile_body<TILE, ACT, X32, O32, PRE, SUM, kGroupNone>(tm_a, tm_b, tm_x, tm_o, p, GroupParams{});
}

template <int TILE, int ACT, bool X32, bool O32, bool PRE, bool SUM>
cudaError_t launch_tile(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tx, const CUtensorMap& to,
                        const LinearParams& given, int sms, cudaStream_t stream) {
  LinearParams p = given;
  using C = LinearCfg<TILE, X32, O32, PRE, SUM>;
  auto kernel = linear_tile_kernel<TILE, ACT, X32, O32, PRE, SUM>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  const int groups = std::min(p.items, sms / C::CG);
  p.kb_q = p.k_blocks / p.splits;
  p.kb_r = p.k_blocks % p.splits;
  p.step_n = groups % p.n_tiles;
  p.step_m = groups / p.n_tiles % p.m_tiles;
  p.step_s = groups / p.n_tiles / p.m_tiles;
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
  return cudaLaunchKernelEx(&cfg, kernel, ta, tb, tx, to, p);
}

template <int TILE, bool X32, bool O32, bool PRE, bool SUM>
cudaError_t by_act(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tx, const CUtensorMap& to,
                   const LinearParams& p, int sms, cudaStream_t st) {
  if (p.act == 1) return launch_tile<TILE, 1, X32, O32, PRE, SUM>(ta, tb, tx, to, p, sms, st);
  if (p.act == 2) return launch_tile<TILE, 2, X32, O32, PRE, SUM>(ta, tb, tx, to, p, sms, st);
  if constexpr (PRE)
    return cudaErrorInvalidValue;  // without an activation the gradient needs no product
  else
    return launch_tile<TILE, 0, X32, O32, PRE, SUM>(ta, tb, tx, to, p, sms, st);
}

template <int TILE>
cudaError_t by_type(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tx, const CUtensorMap& to,
                    const LinearParams& p, int sms, cudaStream_t st) {
  const bool sum = (p.k_blocks + p.splits - 1) / p.splits > p.chunk;  // more than one chunk of k: added in registers
  if (p.pre_grad) {
    if (sum)
      return p.x_f32 ? by_act<TILE, true, false, true, true>(ta, tb, tx, to, p, sms, st)
                     : by_act<TILE, false, false, true, true>(ta, tb, tx, to, p, sms, st);
    return p.x_f32 ? by_act<TILE, true, false, true, false>(ta, tb, tx, to, p, sms, st)
                   : by_act<TILE, false, false, true, false>(ta, tb, tx, to, p, sms, st);
  }
  if (!p.out_f32) return by_act<TILE, false, false, false, false>(ta, tb, tx, to, p, sms, st);
  return sum ? by_act<TILE, true, true, false, true>(ta, tb, tx, to, p, sms, st)
                                                          : by_act<TILE, true, true, false, false>(ta, tb, tx, to, p, sms, st);
}

// ---- the sum of a split product's parts, with the epilogue ----------------------------------------------------------

__device__ __forceinline__ float activate_any(int act, float x) {
  return act == 1 ? activate<1>(x) : act == 2 ? activate<2>(x) : x;
}
// acc at (row, col) through scales, bias, activation and residual, to out.
__device__ __forceinline__ void finish(const LinearParams& p, int64_t row, int col, float acc) {
  if (p.b_scale != nullptr) acc *= p.a_scale[row] * p.b_scale[col];
  if (p.bias != nullptr)
    acc += p.bias_bf16 ? __bfloat162float(static_cast<const bf16*>(p.bias)[col]) : static_cast<const float*>(p.bias)[col];
  acc = activate_any(p.act, acc);
  if (p.x != nullptr) {
    const int64_t at = row * p.ldx + col;
    acc += p.x_f32 ? static_cast<const float*>(p.x)[at] : __bfloat162float(static_cast<const bf16*>(p.x)[at]);
  }
  if (p.out_f32)
    static_cast<float*>(p.out)[row * p.ldo + col] = acc;
  else
    static_cast<bf16*>(p.out)[row * p.ldo + col] = __float2bfloat16_rn(acc);
}

// One column per thread, a row per block row: the parts (in L2, just written) are read once, in split order.
__global__ void __launch_bounds__(256) linear_split_sum_kernel(const float* __restrict__ part, int64_t ldp,
                                                               const LinearParams p) {
  const int64_t row = blockIdx.x;
  const int col = blockIdx.y * 256 + threadIdx.x;
  if (col >= p.n) return;
  float acc = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) acc += part[(s * p.split_rows + row) * ldp + col];
  finish(p, row, col, acc);
}

// ---- few rows ------------------------------------------------------------------------------------------------------

// m <= M rows of a against b [n, k]: a warp per output column, lanes along k, so that b, which is nearly all there is to
// read, streams through wide coalesced loads and a comes from L1. Sums in float32, joined by shuffles.
template <int M, bool FP8, bool WIDE>
__global__ void __launch_bounds__(128) linear_rows_kernel(const uint8_t* __restrict__ a, int64_t lda,
                                                          const uint8_t* __restrict__ b, int64_t ldb,
                                                          const LinearParams p) {
  constexpr int ES = FP8 ? 1 : 2;
  constexpr int V = WIDE ? 16 / ES : 1;
  const int col = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (col >= p.n) return;  // whole warps
  auto widen = [](const uint8_t* src, float (&v)[V]) {
    if constexpr (WIDE) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(src));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (FP8) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t f16x2;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f16x2) : "h"(static_cast<uint16_t>(w[i] >> (16 * h))));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&f16x2));
            v[4 * i + 2 * h] = f.x;
            v[4 * i + 2 * h + 1] = f.y;
          }
        } else {
          const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        }
      }
    } else if constexpr (FP8) {
      uint32_t f16x2;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f16x2) : "h"(static_cast<uint16_t>(__ldg(src))));
      v[0] = __half22float2(*reinterpret_cast<const __half2*>(&f16x2)).x;
    } else {
      v[0] = __bfloat162float(*reinterpret_cast<const bf16*>(src));
    }
  };
  float acc[M];
#pragma unroll
  for (int r = 0; r < M; ++r) acc[r] = 0.f;
  const uint8_t* brow = b + static_cast<int64_t>(col) * ldb * ES;
#pragma unroll 4
  for (int at = lane * V; at < p.k; at += 32 * V) {
    float w[V];
    widen(brow + static_cast<int64_t>(at) * ES, w);
#pragma unroll
    for (int r = 0; r < M; ++r) {
      if (r < p.m) {
        float x[V];
        widen(a + (r * lda + at) * ES, x);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[r] = fmaf(x[e], w[e], acc[r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < M; ++r)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
#pragma unroll
  for (int r = 0; r < M; ++r)
    if (lane == r && r < p.m) finish(p, r, col, acc[r]);
}

template <int M, bool FP8, bool WIDE>
cudaError_t rows_go(const void* a, int64_t lda, const void* b, int64_t ldb, const LinearParams& p, cudaStream_t st) {
  linear_rows_kernel<M, FP8, WIDE><<<(p.n + 3) / 4, 128, 0, st>>>(static_cast<const uint8_t*>(a), lda,
                                                                  static_cast<const uint8_t*>(b), ldb, p);
  return cudaGetLastError();
}
template <int M>
cudaError_t rows_by_type(const void* a, int64_t lda, const void* b, int64_t ldb, bool wide, const LinearParams& p,
                         cudaStream_t st) {
  if (p.fp8) return wide ? rows_go<M, true, true>(a, lda, b, ldb, p, st) : rows_go<M, true, false>(a, lda, b, ldb, p, st);
  return wide ? rows_go<M, false, true>(a, lda, b, ldb, p, st) : rows_go<M, false, false>(a, lda, b, ldb, p, st);
}

// ---- packing and the gradient without an activation ----------------------------------------------------------------

// Rows of any stride and base to rows of whole 16 bytes: a warp per row, a lane gathers 16 bytes and stores them at once
// (the last piece filled up with zeros).
template <class T>
__global__ void __launch_bounds__(256) pack_rows_kernel(const T* __restrict__ src, int64_t lds, T* __restrict__ dst,
                                                        int64_t ldd, int64_t rows, int64_t cols) {
  constexpr int V = 16 / sizeof(T);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const T* from = src + row * lds;
#pragma unroll 2
  for (int64_t j = (threadIdx.x & 31) * V; j < cols; j += 32 * V) {
    __align__(16) T v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = j + e < cols ? from[j + e] : T(0);
    *reinterpret_cast<uint4*>(dst + row * ldd + j) = *reinterpret_cast<const uint4*>(v);
  }
}

// A block takes 32 V columns (lane = V columns) and every gridDim.y-th group of eight rows; partial sums per block in
// float32, added over its eight warps in order.
template <bool X32, int V>
__global__ void __launch_bounds__(256) grad_cast_kernel(const void* __restrict__ x, int64_t ldx, int64_t m, int n,
                                                        bf16* __restrict__ cast, int64_t ldc, float* __restrict__ part) {
  __shared__ float red[8][32 * V + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (blockIdx.x * 32 + lane) * V;
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = 0.f;
  if (col < n) {
#pragma unroll 4
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * 8 + warp; r < m; r += static_cast<int64_t>(gridDim.y) * 8) {
      float v[V];
      if constexpr (V == 8) {
        if constexpr (X32) {
          const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(x) + r * ldx + col);
          const float4 a = __ldg(q), b = __ldg(q + 1);
          v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
          v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const bf16*>(x) + r * ldx + col));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
          }
        }
      } else {
        v[0] = X32 ? static_cast<const float*>(x)[r * ldx + col]
                   : __bfloat162float(static_cast<const bf16*>(x)[r * ldx + col]);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] += v[e];
      if (cast != nullptr) {
        if constexpr (V == 8) {
          uint4 u;
          u.x = pack_bf16(v[0], v[1]);
          u.y = pack_bf16(v[2], v[3]);
          u.z = pack_bf16(v[4], v[5]);
          u.w = pack_bf16(v[6], v[7]);
          *reinterpret_cast<uint4*>(cast + r * ldc + col) = u;
        } else {
          cast[r * ldc + col] = __float2bfloat16_rn(v[0]);
        }
      }
    }
  }
  if (part == nullptr) return;
#pragma unroll
  for (int e = 0; e < V; ++e) red[warp][lane * V + e] = s[e];
  __syncthreads();
  for (int j = threadIdx.x; j < 32 * V; j += 256) {
    const int c = blockIdx.x * 32 * V + j;
    if (c < n) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) t += red[w][j];
      part[static_cast<int64_t>(blockIdx.y) * n + c] = t;
    }
  }
}

}  // namespace

cudaError_t launch_linear_tiles(int tile, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tx,
                                const CUtensorMap& to, const LinearParams& p, int sms, cudaStream_t st) {
  if (tile == kTile256) return by_type<kTile256>(ta, tb, tx, to, p, sms, st);
  if (tile == kTile256Long) return by_type<kTile256Long>(ta, tb, tx, to, p, sms, st);
  if (tile == kTile128) return by_type<kTile128>(ta, tb, tx, to, p, sms, st);
  return by_type<kTile64>(ta, tb, tx, to, p, sms, st);
}

cudaError_t launch_linear_split_sum(const float* part, int64_t ldp, const LinearParams& p, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.m), static_cast<unsigned>((p.n + 255) / 256));
  linear_split_sum_kernel<<<grid, 256, 0, st>>>(part, ldp, p);
  return cudaGetLastError();
}

cudaError_t launch_linear_rows(const void* a, int64_t lda, const void* b, int64_t ldb, bool wide, const LinearParams& p,
                               cudaStream_t st) {
  if (p.m <= 1) return rows_by_type<1>(a, lda, b, ldb, wide, p, st);
  if (p.m <= 2) return rows_by_type<2>(a, lda, b, ldb, wide, p, st);
  if (p.m <= 4) return rows_by_type<4>(a, lda, b, ldb, wide, p, st);
  return rows_by_type<kLinearRowsMax>(a, lda, b, ldb, wide, p, st);
}

cudaError_t launch_pack_rows(const void* src, int64_t lds, void* dst, int64_t ldd, int64_t rows, int64_t cols, int es,
                             cudaStream_t st) {
  const int64_t blocks = (rows + 7) / 8;
  if (blocks == 0) return cudaSuccess;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  if (es == 1)
    pack_rows_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(static_cast<const uint8_t*>(src), lds,
                                                                    static_cast<uint8_t*>(dst), ldd, rows, cols);
  else
    pack_rows_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(static_cast<const uint16_t*>(src), lds,
                                                                    static_cast<uint16_t*>(dst), ldd, rows, cols);
  return cudaGetLastError();
}

int grad_cast_blocks(int64_t m, int n, int sms) {
  const int64_t across = (n + 255) / 256;
  const int64_t want = std::max<int64_t>(1, 8 * static_cast<int64_t>(sms) / across);
  return static_cast<int>(std::min<int64_t>(want, std::max<int64_t>(1, (m + 7) / 8)));
}

cudaError_t launch_grad_cast(const void* x, bool x_f32, int64_t ldx, int64_t m, int n, void* cast, int64_t ldc,
                             float* part, int blocks, bool wide, cudaStream_t st) {
  const int v = wide ? 8 : 1;
  const dim3 grid(static_cast<unsigned>((n + 32 * v - 1) / (32 * v)), static_cast<unsigned>(blocks));
  auto* c = static_cast<bf16*>(cast);
  if (x_f32) {
    if (wide) grad_cast_kernel<true, 8><<<grid, 256, 0, st>>>(x, ldx, m, n, c, ldc, part);
    else grad_cast_kernel<true, 1><<<grid, 256, 0, st>>>(x, ldx, m, n, c, ldc, part);
  } else {
    if (wide) grad_cast_kernel<false, 8><<<grid, 256, 0, st>>>(x, ldx, m, n, c, ldc, part);
    else grad_cast_kernel<false, 1><<<grid, 256, 0, st>>>(x, ldx, m, n, c, ldc, part);
  }
  return cudaGetLastError();
}

cudaError_t take_linear_error(unsigned int* word) {
  cudaError_t e = cudaMemcpyFromSymbol(word, g_device_error, sizeof(*word));
  if (e != cudaSuccess) return e;
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
}

}  // namespace fwn
