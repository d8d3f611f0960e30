// Root-mean-square norm of a residual stream, with the residual's addition, an 8-bit output with scales, and its
// gradient:
//   s = x + residual,  rstd = 1 / sqrt(mean(s^2) + eps),  h = s rstd weight
// (x, s float32 or bf16, residual and weight float32, bf16 or absent, h bf16, float32, or e4m3 with one float32 scale
// per row, scale = max |h| / 448, h = scale * value). Sums are float32; s is normalised unrounded and rounded once,
// where it is stored.
//
// Bound: HBM. A row is read once, kept in registers (at most 32 values per thread) through the sum of squares (and the
// row maximum of the 8-bit output) and written once. A row of up to 1,024 values belongs to one warp, of up to 8,192
// to a block of 256 threads, of up to 16,384 to one of 1,024: the smallest group that holds the row in registers
// needs the fewest exchanges. Rows whose width and addresses allow it move as 8 values per thread (16 bytes of bf16,
// 32 of float32, the widest accesses of sm_100); others (odd widths) one value per thread, still coalesced.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "rms.cuh"

namespace fwn {

namespace {

using bf16 = __nv_bfloat16;
struct none_t {};
struct e4m3_t { uint8_t v; };

template <class T> constexpr bool is_none = false;
template <> constexpr bool is_none<none_t> = true;

// V values at p as float32. V = 8: one 16-byte (bf16) or 32-byte (float32) access; V = 1: one element.
template <int V>
__device__ __forceinline__ void load_vals(const float* p, float (&v)[V]) {
  if constexpr (V == 8) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "l"(p));
  } else {
    v[0] = __ldg(p);
  }
}
template <int V>
__device__ __forceinline__ void load_vals(const bf16* p, float (&v)[V]) {
  if constexpr (V == 8) {
    uint32_t u[4];
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3])
                 : "l"(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
    v[0] = __bfloat162float(p[0]);
  }
}

template <int V>
__device__ __forceinline__ void store_vals(float* p, const float (&v)[V]) {
  if constexpr (V == 8) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                 "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
  } else {
    p[0] = v[0];
  }
}
template <int V>
__device__ __forceinline__ void store_vals(bf16* p, const float (&v)[V]) {
  if constexpr (V == 8) {
    uint4 u;
    uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = u;
  } else {
    p[0] = __float2bfloat16_rn(v[0]);
  }
}
// Round to nearest even, saturating at +-448; NaN stays NaN.
__device__ __forceinline__ uint32_t pack_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
template <int V>
__device__ __forceinline__ void store_vals(e4m3_t* p, const float (&v)[V]) {
  if constexpr (V == 8) {
    uint2 u;
    u.x = pack_e4m3x2(v[0], v[1]) | (pack_e4m3x2(v[2], v[3]) << 16);
    u.y = pack_e4m3x2(v[4], v[5]) | (pack_e4m3x2(v[6], v[7]) << 16);
    *reinterpret_cast<uint2*>(p) = u;
  } else {
    p[0].v = static_cast<uint8_t>(pack_e4m3x2(v[0], 0.f) & 0xFFu);
  }
}

// V weights (a row every row reads again: kept in L1).
template <int V>
__device__ __forceinline__ void load_weight(const void* w, bool w_bf16, int at, float (&v)[V]) {
  if (w_bf16) {
    const bf16* p = static_cast<const bf16*>(w) + at;
    if constexpr (V == 8) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&q[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    } else {
      v[0] = __bfloat162float(p[0]);
    }
  } else {
    const float* p = static_cast<const float*>(w) + at;
    if constexpr (V == 8) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      v[0] = __ldg(p);
    }
  }
}

// Maximum that keeps a NaN, so that a row with one gets a NaN scale.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sum (or NaN-keeping maximum) over the TPR threads of a row, the same in each. `red` holds one value per warp and is
// used once per call site and row, so the block form needs a barrier before the next row's use (two alternate).
template <int TPR, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? max_nan(v, u) : v + u;
  }
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[threadIdx.x & (TPR / 32 - 1)];
#pragma unroll
    for (int o = TPR / 64; o > 0; o >>= 1) {
      const float u = __shfl_xor_sync(0xffffffffu, v, o);
      v = MAX ? max_nan(v, u) : v + u;
    }
  }
  return v;
}

// Index of a thread's i-th group of V values, and whether it lies in the row.
template <int TPR, int V>
__device__ __forceinline__ int val_at(int i) {
  const int t = TPR == 32 ? (threadIdx.x & 31) : threadIdx.x;
  return (i * TPR + t) * V;
}

constexpr float kE4m3Max = 448.f;
// A row whose largest value is below this has scale 0 and values 0 (its scale's reciprocal would leave float32).
constexpr float kTinyRow = 7.8886090522101181e-31f;  // 2^-100

// TPR threads per row (32: a warp, eight rows per block of 256; else the block), NV groups of V values per thread.
template <class X, class R, class O, int TPR, int V, int NV>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, TPR == 1024 ? 1 : 2) rms_norm_kernel(const RmsParams p) {
  __shared__ float red[2][32];
  const int64_t row = TPR == 32 ? (static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5))
                                : static_cast<int64_t>(blockIdx.x);
  if (row >= p.rows) return;  // whole warps leave together
  const X* x = static_cast<const X*>(p.x) + row * p.x_stride;
  float s[NV][V];
  float r[is_none<R> ? 1 : NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = val_at<TPR, V>(i);
#pragma unroll
    for (int e = 0; e < V; ++e) s[i][e] = 0.f;
    if (at < p.d) load_vals(x + at, s[i]);
    if constexpr (!is_none<R>) {
#pragma unroll
      for (int e = 0; e < V; ++e) r[i][e] = 0.f;
      if (at < p.d) load_vals(static_cast<const R*>(p.residual) + row * p.residual_stride + at, r[i]);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if constexpr (!is_none<R>) {
#pragma unroll
      for (int e = 0; e < V; ++e) s[i][e] += r[i][e];
      const int at = val_at<TPR, V>(i);
      if (at < p.d) store_vals(static_cast<X*>(p.x_out) + row * p.d + at, s[i]);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) ss = fmaf(s[i][e], s[i][e], ss);
  }
  float rstd = 1.f;
  if (p.normalize) {
    ss = row_reduce<TPR, false>(ss, red[0]);
    rstd = rsqrtf(ss / static_cast<float>(p.d) + p.eps);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = val_at<TPR, V>(i);
    if (p.weight != nullptr && at < p.d) {
      float w[V];
      load_weight(p.weight, p.weight_bf16, at, w);
#pragma unroll
      for (int e = 0; e < V; ++e) s[i][e] = s[i][e] * rstd * w[e];
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) s[i][e] *= rstd;
    }
  }
  if constexpr (sizeof(O) == 1) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) m = max_nan(m, fabsf(s[i][e]));
    m = row_reduce<TPR, true>(m, red[1]);
    const bool tiny = m < kTinyRow;  // false for NaN, which the scale and the values keep
    const float inv = tiny ? 0.f : kE4m3Max / m;
    if ((TPR == 32 ? (threadIdx.x & 31) : threadIdx.x) == 0) p.scale[row] = tiny ? 0.f : m / kE4m3Max;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) s[i][e] *= inv;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = val_at<TPR, V>(i);
    if (at < p.d) store_vals(static_cast<O*>(p.out) + row * p.d + at, s[i]);
  }
}

// Gradient, with g = dh weight, s the normalised row (x, or x + residual), ds the gradient of the stored sum:
//   dx = rstd g - s rstd^3 mean(g s) + ds,  d_residual = dx,  dweight = sum over rows of dh s rstd.
// A group of TPR threads walks rows (grid-stride); its columns' share of dweight stays in registers and leaves as one
// row of partials per block (the warps of a block are added through shared memory), summed in order by
// rms_weight_sum_kernel: no atomics, the same bits every time. Both row sums go through one pair of exchanges.
template <class X, class R, class G, int TPR, int V, int NV>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, TPR == 1024 ? 1 : 2) rms_norm_bwd_kernel(const RmsBwdParams p) {
  constexpr int kWarps = TPR == 32 ? 8 : 1;
  extern __shared__ float part_smem[];  // TPR == 32 with a weight: 8 rows of d
  __shared__ float red[4][32];
  const int64_t first = TPR == 32 ? static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = TPR == 32 ? static_cast<int64_t>(gridDim.x) * 8 : gridDim.x;
  float dw[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) dw[i][e] = 0.f;
  int flip = 0;
  for (int64_t row = first; row < p.rows; row += step, flip ^= 2) {
    float s[NV][V], g[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = val_at<TPR, V>(i);
#pragma unroll
      for (int e = 0; e < V; ++e) s[i][e] = g[i][e] = 0.f;
      if (at < p.d) {
        load_vals(static_cast<const X*>(p.x) + row * p.x_stride + at, s[i]);
        load_vals(static_cast<const G*>(p.dh) + row * p.d + at, g[i]);
        if constexpr (!is_none<R>) {
          if (p.residual != nullptr) {
            float r[V];
            load_vals(static_cast<const R*>(p.residual) + row * p.residual_stride + at, r);
#pragma unroll
            for (int e = 0; e < V; ++e) s[i][e] += r[e];
          }
        }
      }
    }
    float ss = 0.f, sg = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = val_at<TPR, V>(i);
      if (p.weight != nullptr && at < p.d) {
        float w[V];
        load_weight(p.weight, p.weight_bf16, at, w);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          ss = fmaf(s[i][e], s[i][e], ss);
          sg = fmaf(g[i][e] * w[e], s[i][e], sg);
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          ss = fmaf(s[i][e], s[i][e], ss);
          sg = fmaf(g[i][e], s[i][e], sg);
        }
      }
    }
    ss = row_reduce<TPR, false>(ss, red[flip]);
    sg = row_reduce<TPR, false>(sg, red[flip + 1]);
    const float rstd = rsqrtf(ss / static_cast<float>(p.d) + p.eps);
    const float c = sg / static_cast<float>(p.d) * rstd * rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = val_at<TPR, V>(i);
      if (at >= p.d) continue;
      float dx[V];
      if (p.weight != nullptr) {
        float w[V];
        load_weight(p.weight, p.weight_bf16, at, w);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          dw[i][e] = fmaf(g[i][e], s[i][e] * rstd, dw[i][e]);
          dx[e] = rstd * (g[i][e] * w[e] - s[i][e] * c);
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) dx[e] = rstd * (g[i][e] - s[i][e] * c);
      }
      if (p.ds != nullptr) {
        float ds[V];
        load_vals(static_cast<const X*>(p.ds) + row * p.d + at, ds);
#pragma unroll
        for (int e = 0; e < V; ++e) dx[e] += ds[e];
      }
      if (p.dx != nullptr) store_vals(static_cast<X*>(p.dx) + row * p.d + at, dx);
      if constexpr (!is_none<R>) {
        if (p.dr != nullptr) store_vals(static_cast<R*>(p.dr) + row * p.d + at, dx);
      }
    }
  }
  if (p.part == nullptr) return;
  if constexpr (kWarps > 1) {
    float* mine = part_smem + (threadIdx.x >> 5) * p.d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = val_at<TPR, V>(i);
      if (at < p.d) {
#pragma unroll
        for (int e = 0; e < V; ++e) mine[at + e] = dw[i][e];
      }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < p.d; j += blockDim.x) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) t += part_smem[w * p.d + j];
      p.part[static_cast<int64_t>(blockIdx.x) * p.d + j] = t;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = val_at<TPR, V>(i);
      if (at < p.d) {
#pragma unroll
        for (int e = 0; e < V; ++e) p.part[static_cast<int64_t>(blockIdx.x) * p.d + at + e] = dw[i][e];
      }
    }
  }
}

// out[j] = sum over r of part[r, j], j < d: a block takes 32 columns, its 32 warps every 32nd row (eight loads in
// flight each), and their sums are added in order.
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ part, int64_t rows, int d,
                                                           void* __restrict__ out, bool out_bf16) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (j < d) {
#pragma unroll 8
    for (int64_t r = warp; r < rows; r += 32) t += part[r * d + j];
  }
  red[warp][lane] = t;
  __syncthreads();
  t = red[lane][warp];  // column `warp` of the block, the sums of its warps across the lanes
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  const int c = blockIdx.x * 32 + warp;
  if (lane == 0 && c < d) {
    if (out_bf16)
      static_cast<bf16*>(out)[c] = __float2bfloat16_rn(t);
    else
      static_cast<float*>(out)[c] = t;
  }
}

template <class X, class R, class O, int TPR, int V, int NV>
cudaError_t go(const RmsParams& p, cudaStream_t st) {
  const int64_t blocks = TPR == 32 ? (p.rows + 7) / 8 : p.rows;
  rms_norm_kernel<X, R, O, TPR, V, NV><<<static_cast<unsigned>(blocks), TPR == 32 ? 256 : TPR, 0, st>>>(p);
  return cudaGetLastError();
}
template <class X, class R, class O, int V>
cudaError_t by_width(const RmsParams& p, cudaStream_t st) {
  constexpr int U = 8 / V;  // groups per 8 values
  if (p.d <= 256) return go<X, R, O, 32, V, U>(p, st);
  if (p.d <= 512) return go<X, R, O, 32, V, 2 * U>(p, st);
  if (p.d <= 1024) return go<X, R, O, 32, V, 4 * U>(p, st);
  if (p.d <= 2048) return go<X, R, O, 256, V, U>(p, st);
  if (p.d <= 4096) return go<X, R, O, 256, V, 2 * U>(p, st);
  if (p.d <= 8192) return go<X, R, O, 256, V, 4 * U>(p, st);
  return go<X, R, O, 1024, V, 2 * U>(p, st);
}
template <class X, class R>
cudaError_t by_out(const RmsParams& p, cudaStream_t st) {
  switch (p.out_type) {
    case kRmsBf16: return p.wide ? by_width<X, R, bf16, 8>(p, st) : by_width<X, R, bf16, 1>(p, st);
    case kRmsF32: return p.wide ? by_width<X, R, float, 8>(p, st) : by_width<X, R, float, 1>(p, st);
    default: return p.wide ? by_width<X, R, e4m3_t, 8>(p, st) : by_width<X, R, e4m3_t, 1>(p, st);
  }
}
template <class X>
cudaError_t by_residual(const RmsParams& p, cudaStream_t st) {
  if (p.residual == nullptr) return by_out<X, none_t>(p, st);
  return p.residual_bf16 ? by_out<X, bf16>(p, st) : by_out<X, float>(p, st);
}

template <class X, class R, class G, int TPR, int V, int NV>
cudaError_t go_bwd(const RmsBwdParams& p, int blocks, cudaStream_t st) {
  const size_t smem = TPR == 32 && p.part != nullptr ? 8 * sizeof(float) * static_cast<size_t>(p.d) : 0;
  rms_norm_bwd_kernel<X, R, G, TPR, V, NV><<<blocks, TPR == 32 ? 256 : TPR, smem, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.part == nullptr) return e;
  return launch_column_sum(p.part, blocks, p.d, p.dw, p.dw_bf16, st);
}
template <class X, class R, class G, int V>
cudaError_t bwd_by_width(const RmsBwdParams& p, int blocks, cudaStream_t st) {
  constexpr int U = 8 / V;
  if (p.d <= 256) return go_bwd<X, R, G, 32, V, U>(p, blocks, st);
  if (p.d <= 512) return go_bwd<X, R, G, 32, V, 2 * U>(p, blocks, st);
  if (p.d <= 1024) return go_bwd<X, R, G, 32, V, 4 * U>(p, blocks, st);
  if (p.d <= 2048) return go_bwd<X, R, G, 256, V, U>(p, blocks, st);
  if (p.d <= 4096) return go_bwd<X, R, G, 256, V, 2 * U>(p, blocks, st);
  if (p.d <= 8192) return go_bwd<X, R, G, 256, V, 4 * U>(p, blocks, st);
  return go_bwd<X, R, G, 1024, V, 2 * U>(p, blocks, st);
}
template <class X, class R>
cudaError_t bwd_by_grad(const RmsBwdParams& p, int blocks, cudaStream_t st) {
  if (p.dh_bf16) return p.wide ? bwd_by_width<X, R, bf16, 8>(p, blocks, st) : bwd_by_width<X, R, bf16, 1>(p, blocks, st);
  return p.wide ? bwd_by_width<X, R, float, 8>(p, blocks, st) : bwd_by_width<X, R, float, 1>(p, blocks, st);
}
template <class X>
cudaError_t bwd_by_residual(const RmsBwdParams& p, int blocks, cudaStream_t st) {
  if (p.residual == nullptr && p.dr == nullptr) return bwd_by_grad<X, none_t>(p, blocks, st);
  return p.residual_bf16 ? bwd_by_grad<X, bf16>(p, blocks, st) : bwd_by_grad<X, float>(p, blocks, st);
}

}  // namespace

cudaError_t launch_rms_norm(const RmsParams& p, cudaStream_t st) {
  if (p.rows == 0) return cudaSuccess;
  return p.x_bf16 ? by_residual<bf16>(p, st) : by_residual<float>(p, st);
}

// Blocks of the gradient's kernel: two (warp per row) per SM are resident at the widths that need the most registers;
// enough rows per block remain to spread the cost of its row of partials.
int rms_bwd_blocks(int64_t rows, int d, int sms) {
  const int64_t most = d <= 1024 ? (rows + 7) / 8 : rows;
  const int64_t resident = static_cast<int64_t>(sms) * (d <= 1024 ? 2 : d <= 8192 ? 2 : 1);
  return static_cast<int>(most < resident ? most : resident);
}

cudaError_t launch_rms_norm_bwd(const RmsBwdParams& p, int blocks, cudaStream_t st) {
  if (p.rows == 0) {
    if (p.part == nullptr) return cudaSuccess;
    return launch_column_sum(p.part, 0, p.d, p.dw, p.dw_bf16, st);
  }
  return p.x_bf16 ? bwd_by_residual<bf16>(p, blocks, st) : bwd_by_residual<float>(p, blocks, st);
}

cudaError_t launch_column_sum(const float* part, int64_t rows, int d, void* out, bool out_bf16, cudaStream_t st) {
  column_sum_kernel<<<(d + 31) / 32, 1024, 0, st>>>(part, rows, d, out, out_bf16);
  return cudaGetLastError();
}

}  // namespace fwn
