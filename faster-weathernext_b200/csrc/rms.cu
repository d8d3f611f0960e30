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
// needs the fewest exchanges. Three ways to lay a row over its threads:
//   kWide    8 values per thread and access (16 bytes of bf16, 32 of float32, the widest accesses of sm_100): widths
//            and strides that are multiples of 8;
//   kShift   the same accesses for rows of any width that follow one another without gaps: groups of 8 start at the
//            aligned address before the row, and only the two that its ends cut go by single values. A group of threads
//            takes rows eight apart, whose starts are off alike, so that a thread keeps its columns (its weights, its
//            share of the weight's gradient) from row to row, and the next row's loads are issued before the work on
//            one. 10,242 x 1,001 bf16 with a bf16 residual, forward / backward: kScalar 41 / 165 us, kShift 22 / 35;
//   kScalar  one value per thread and access: other strides and addresses.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "rms.cuh"

namespace fwn {

namespace {

using bf16 = __nv_bfloat16;
struct none_t {};
struct e4m3_t { uint8_t v; };

template <class T> constexpr bool is_none = false;
template <> constexpr bool is_none<none_t> = true;

// V values of type T as they were loaded. V = 8: one 16-byte (bf16) or 32-byte (float32) access; V = 1: one element.
template <class T, int V>
struct Raw {
  uint32_t u[V == 1 ? 1 : V * sizeof(T) / 4];
};
template <int V>
__device__ __forceinline__ void load_raw(const float* p, Raw<float, V>& r) {
  if constexpr (V == 8) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r.u[0]), "=r"(r.u[1]), "=r"(r.u[2]), "=r"(r.u[3]), "=r"(r.u[4]), "=r"(r.u[5]), "=r"(r.u[6]), "=r"(r.u[7])
                 : "l"(p));
  } else {
    r.u[0] = __float_as_uint(__ldg(p));
  }
}
template <int V>
__device__ __forceinline__ void load_raw(const bf16* p, Raw<bf16, V>& r) {
  if constexpr (V == 8) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.u[0]), "=r"(r.u[1]), "=r"(r.u[2]), "=r"(r.u[3])
                 : "l"(p));
  } else {
    r.u[0] = __ldg(reinterpret_cast<const unsigned short*>(p));
  }
}
template <int V>
__device__ __forceinline__ float raw_at(const Raw<float, V>& r, int e) { return __uint_as_float(r.u[e]); }
template <int V>
__device__ __forceinline__ float raw_at(const Raw<bf16, V>& r, int e) {
  return __uint_as_float(e & 1 ? r.u[e / 2] & 0xFFFF0000u : r.u[e / 2] << 16);
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

enum RowMode { kScalar = 0, kWide = 1, kShift = 2 };

// Column of a thread's i-th group of V values; `off` (kShift) is how far the row starts past an aligned address.
template <int TPR, int V>
__device__ __forceinline__ int group_at(int i, int off) {
  const int t = TPR == 32 ? (threadIdx.x & 31) : threadIdx.x;
  return (i * TPR + t) * V - off;
}
// The group of values from column j of the row at p. `more`: rows follow, so that a group which the row's end cuts may be
// read whole (kShift: what lies before a row is the row before); the last row's goes by single values.
template <int MODE, class T, int V>
__device__ __forceinline__ void load_group(const T* p, int j, int d, bool more, Raw<T, V>& r) {
  constexpr int W = sizeof(r.u) / 4;
#pragma unroll
  for (int i = 0; i < W; ++i) r.u[i] = 0;
  if constexpr (MODE == kShift) {
    if (j < d && (more || j + V <= d)) {
      load_raw(p + j, r);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (j + e >= 0 && j + e < d) {
          Raw<T, 1> one;
          load_raw(p + j + e, one);
          if constexpr (sizeof(T) == 4)
            r.u[e] = one.u[0];
          else
            r.u[e / 2] |= one.u[0] << (e & 1 ? 16 : 0);
        }
      }
    }
  } else {
    if (j < d) load_raw(p + j, r);
  }
}
// Its values; columns outside [0, d) are 0.
template <int MODE, class T, int V>
__device__ __forceinline__ void expand(const Raw<T, V>& r, int j, int d, float (&v)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    v[e] = raw_at(r, e);
    if constexpr (MODE == kShift) v[e] = j + e >= 0 && j + e < d ? v[e] : 0.f;
  }
}
template <int MODE, class T, int V>
__device__ __forceinline__ void store_group(T* p, int j, int d, const float (&v)[V]) {
  if constexpr (MODE == kShift) {
    if (j >= 0 && j + V <= d) {
      store_vals(p + j, v);
    } else if (j < d && j + V > 0) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float one[1] = {v[e]};
        if (j + e >= 0 && j + e < d) store_vals(p + j + e, one);
      }
    }
  } else {
    if (j < d) store_vals(p + j, v);
  }
}
template <int MODE, int V>
__device__ __forceinline__ void weight_group(const void* w, bool w_bf16, int j, int d, float (&v)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = 0.f;
  if constexpr (MODE == kShift) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float one[1];
      if (j + e >= 0 && j + e < d) {
        load_weight(w, w_bf16, j + e, one);
        v[e] = one[0];
      }
    }
  } else {
    if (j < d) load_weight(w, w_bf16, j, v);
  }
}

constexpr float kE4m3Max = 448.f;
// A row whose largest value is below this has scale 0 and values 0 (its scale's reciprocal would leave float32).
constexpr float kTinyRow = 7.8886090522101181e-31f;  // 2^-100

// TPR threads per row (32: a warp, eight rows per block of 256; else the block), NV groups of V values per thread. The
// grid covers the rows, or (kShift) a multiple of eight blocks walks them.
template <class X, class R, class O, int TPR, int MODE, int NV>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, TPR == 1024 ? 1 : 2) rms_norm_kernel(const RmsParams p) {
  constexpr int V = MODE == kScalar ? 1 : 8;
  __shared__ float red[4][32];
  const int64_t first = TPR == 32 ? static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (TPR == 32 ? 8 : 1);
  const int off = MODE == kShift ? static_cast<int>(first * p.d & 7) : 0;  // of all this group's rows
  const int d = p.d;
  float w[MODE == kShift ? NV : 1][V];
  if constexpr (MODE == kShift) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (p.weight != nullptr) {
        weight_group<MODE>(p.weight, p.weight_bf16, group_at<TPR, V>(i, off), d, w[i]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) w[i][e] = 1.f;
      }
    }
  }
  using RR = std::conditional_t<is_none<R>, float, R>;
  constexpr int NR = is_none<R> ? 1 : NV;
  constexpr bool kAhead = MODE == kShift;  // the next row is on its way while one is worked on
  Raw<X, V> xs[kAhead ? NV : 1];
  Raw<RR, V> rs[kAhead ? NR : 1];
  auto fetch = [&](int64_t row, int i, Raw<X, V>& a, Raw<RR, V>& b) {
    const int j = group_at<TPR, V>(i, off);
    load_group<MODE>(static_cast<const X*>(p.x) + row * p.x_stride, j, d, row + 1 < p.rows, a);
    if constexpr (!is_none<R>)
      load_group<MODE>(static_cast<const R*>(p.residual) + row * p.residual_stride, j, d, row + 1 < p.rows, b);
  };
  auto fetch_row = [&](int64_t row) {
    if (!kAhead || row >= p.rows) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) fetch(row, i, xs[kAhead ? i : 0], rs[kAhead && !is_none<R> ? i : 0]);
  };
  fetch_row(first);
  int flip = 0;
  for (int64_t row = first; row < p.rows; row += step, flip ^= 2) {  // whole warps (blocks) leave together
    float s[NV][V], r[NR][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = group_at<TPR, V>(i, off);
      Raw<X, V> a;
      Raw<RR, V> b;
      if constexpr (kAhead) {
        a = xs[i];
        b = rs[is_none<R> ? 0 : i];
      } else {
        fetch(row, i, a, b);
      }
      expand<MODE>(a, j, d, s[i]);
      if constexpr (!is_none<R>) expand<MODE>(b, j, d, r[i]);
    }
    fetch_row(row + step);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (!is_none<R>) {
#pragma unroll
        for (int e = 0; e < V; ++e) s[i][e] += r[i][e];
        store_group<MODE>(static_cast<X*>(p.x_out) + row * d, group_at<TPR, V>(i, off), d, s[i]);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) ss = fmaf(s[i][e], s[i][e], ss);
    }
    float rstd = 1.f;
    if (p.normalize) {
      ss = row_reduce<TPR, false>(ss, red[flip]);
      rstd = rsqrtf(ss / static_cast<float>(d) + p.eps);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (MODE == kShift) {
#pragma unroll
        for (int e = 0; e < V; ++e) s[i][e] = s[i][e] * rstd * w[i][e];
      } else if (p.weight != nullptr) {
        weight_group<MODE>(p.weight, p.weight_bf16, group_at<TPR, V>(i, off), d, w[0]);
#pragma unroll
        for (int e = 0; e < V; ++e) s[i][e] = s[i][e] * rstd * w[0][e];
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
      m = row_reduce<TPR, true>(m, red[flip + 1]);
      const bool tiny = m < kTinyRow;  // false for NaN, which the scale and the values keep
      const float inv = tiny ? 0.f : kE4m3Max / m;
      if ((TPR == 32 ? (threadIdx.x & 31) : threadIdx.x) == 0) p.scale[row] = tiny ? 0.f : m / kE4m3Max;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) s[i][e] *= inv;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) store_group<MODE>(static_cast<O*>(p.out) + row * d, group_at<TPR, V>(i, off), d, s[i]);
  }
}

// Blocks of the gradient's kernel that an SM holds, by the threads of a row and the values of a thread: five arrays of
// values and some 30 registers a thread.
constexpr int bwd_resident(int tpr, int values) {
  return tpr == 1024 ? 1 : tpr == 128 ? 4 : values <= 8 && tpr == 32 ? 3 : 2;
}

// Gradient, with g = dh weight, s the normalised row (x, or x + residual), ds the gradient of the stored sum:
//   dx = rstd g - s rstd^3 mean(g s) + ds,  d_residual = dx,  dweight = sum over rows of dh s rstd.
// A group of TPR threads walks rows (grid-stride); its columns' share of dweight stays in registers and leaves as one
// row of partials per block (the warps of a block are added through shared memory), summed in order by
// column_sum_kernel: no atomics, the same bits every time. All of a row's loads are issued before its sums are needed.
template <class X, class R, class G, int TPR, int MODE, int NV>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, bwd_resident(TPR, NV * (MODE == kScalar ? 1 : 8)))
    rms_norm_bwd_kernel(const RmsBwdParams p) {
  constexpr int V = MODE == kScalar ? 1 : 8;
  extern __shared__ float part_smem[];  // TPR == 32 with a weight: 8 rows of d
  __shared__ float red[4][32];
  const int64_t first = TPR == 32 ? static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (TPR == 32 ? 8 : 1);
  const int off = MODE == kShift ? static_cast<int>(first * p.d & 7) : 0;
  const int d = p.d;
  float w[NV][V], dw[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (p.weight != nullptr) {
      weight_group<MODE>(p.weight, p.weight_bf16, group_at<TPR, V>(i, off), d, w[i]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) w[i][e] = 1.f;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) dw[i][e] = 0.f;
  }
  using RR = std::conditional_t<is_none<R>, float, R>;
  constexpr bool kAhead = MODE == kShift && NV == 1;  // the next row is on its way while one is worked on
  struct Loads {
    Raw<X, V> x, ds;
    Raw<G, V> g;
    Raw<RR, V> r;
  };
  Loads next;
  auto fetch = [&](int64_t row, int i, Loads& l) {
    const bool more = row + 1 < p.rows;
    const int j = group_at<TPR, V>(i, off);
    load_group<MODE>(static_cast<const X*>(p.x) + row * p.x_stride, j, d, more, l.x);
    load_group<MODE>(static_cast<const G*>(p.dh) + row * d, j, d, more, l.g);
    if (p.ds != nullptr) load_group<MODE>(static_cast<const X*>(p.ds) + row * d, j, d, more, l.ds);
    if constexpr (!is_none<R>) {
      if (p.residual != nullptr)
        load_group<MODE>(static_cast<const R*>(p.residual) + row * p.residual_stride, j, d, more, l.r);
    }
  };
  if (kAhead && first < p.rows) fetch(first, 0, next);
  int flip = 0;
  for (int64_t row = first; row < p.rows; row += step, flip ^= 2) {
    float s[NV][V], g[NV][V], ds[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = group_at<TPR, V>(i, off);
      Loads l;
      if constexpr (kAhead) l = next; else fetch(row, i, l);
      expand<MODE>(l.x, j, d, s[i]);
      expand<MODE>(l.g, j, d, g[i]);
      if (p.ds != nullptr) {
        expand<MODE>(l.ds, j, d, ds[i]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) ds[i][e] = 0.f;
      }
      if constexpr (!is_none<R>) {
        if (p.residual != nullptr) {
          float r[V];
          expand<MODE>(l.r, j, d, r);
#pragma unroll
          for (int e = 0; e < V; ++e) s[i][e] += r[e];
        }
      }
    }
    if (kAhead && row + step < p.rows) fetch(row + step, 0, next);
    float ss = 0.f, sg = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        ss = fmaf(s[i][e], s[i][e], ss);
        sg = fmaf(g[i][e] * w[i][e], s[i][e], sg);
      }
    }
    ss = row_reduce<TPR, false>(ss, red[flip]);
    sg = row_reduce<TPR, false>(sg, red[flip + 1]);
    const float rstd = rsqrtf(ss / static_cast<float>(d) + p.eps);
    const float c = sg / static_cast<float>(d) * rstd * rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = group_at<TPR, V>(i, off);
      float dx[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        dw[i][e] = fmaf(g[i][e], s[i][e] * rstd, dw[i][e]);
        dx[e] = fmaf(rstd, g[i][e] * w[i][e] - s[i][e] * c, ds[i][e]);
      }
      if (p.dx != nullptr) store_group<MODE>(static_cast<X*>(p.dx) + row * d, j, d, dx);
      if constexpr (!is_none<R>) {
        if (p.dr != nullptr) store_group<MODE>(static_cast<R*>(p.dr) + row * d, j, d, dx);
      }
    }
  }
  if (p.part == nullptr) return;
  float* mine = TPR == 32 ? part_smem + (threadIdx.x >> 5) * d : p.part + static_cast<int64_t>(blockIdx.x) * d;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = group_at<TPR, V>(i, off);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (j + e >= 0 && j + e < d) mine[j + e] = dw[i][e];
  }
  if constexpr (TPR == 32) {
    __syncthreads();
    for (int j = threadIdx.x; j < d; j += blockDim.x) {
      float t = 0.f;
#pragma unroll
      for (int v = 0; v < 8; ++v) t += part_smem[v * d + j];
      p.part[static_cast<int64_t>(blockIdx.x) * d + j] = t;
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

// Calls f with the threads per row and the groups per thread that hold `room` values. LEAN: at most 16 values per thread
// up to 8,192 of a row (the gradient keeps five arrays of them, kShift three).
template <int MODE, bool LEAN, class F>
cudaError_t by_width(int room, F f) {
  using std::integral_constant;
  if constexpr (MODE == kScalar) {
    if (room <= 2048) return f(integral_constant<int, 256>(), integral_constant<int, 8>());
    if (room <= 4096) return f(integral_constant<int, 256>(), integral_constant<int, 16>());
    return f(integral_constant<int, 1024>(), integral_constant<int, 16>());
  } else {
    if (room <= 256) return f(integral_constant<int, 32>(), integral_constant<int, 1>());
    if (room <= 512) return f(integral_constant<int, 32>(), integral_constant<int, 2>());
    if constexpr (LEAN) {
      if (room <= 1024) return f(integral_constant<int, 128>(), integral_constant<int, 1>());
    } else {
      if (room <= 1024) return f(integral_constant<int, 32>(), integral_constant<int, 4>());
    }
    if (room <= 2048) return f(integral_constant<int, 256>(), integral_constant<int, 1>());
    if (room <= 4096) return f(integral_constant<int, 256>(), integral_constant<int, 2>());
    if constexpr (LEAN) {
      if (room <= 8192) return f(integral_constant<int, 1024>(), integral_constant<int, 1>());
    } else {
      if (room <= 8192) return f(integral_constant<int, 256>(), integral_constant<int, 4>());
    }
    return f(integral_constant<int, 1024>(), integral_constant<int, 2>());
  }
}
int room_of(int mode, int d) { return mode == kShift ? d + 7 : d; }

template <class X, class R, class O, int MODE>
cudaError_t go(const RmsParams& p, cudaStream_t st) {
  return by_width<MODE, MODE == kShift>(room_of(MODE, p.d), [&](auto tpr, auto nv) {
    constexpr int TPR = decltype(tpr)::value;
    int64_t blocks = TPR == 32 ? (p.rows + 7) / 8 : p.rows;
    if (MODE == kShift) {
      // A multiple of eight, several rows each: the weights are read once per group of threads.
      const int64_t resident = static_cast<int64_t>(p.sms) * (TPR == 1024 ? 1 : TPR == 128 ? 6 : 2);
      blocks = std::min(blocks, resident);
      if (TPR != 32) blocks = (blocks + 7) / 8 * 8;
    }
    rms_norm_kernel<X, R, O, TPR, MODE, decltype(nv)::value>
        <<<static_cast<unsigned>(blocks), TPR == 32 ? 256 : TPR, 0, st>>>(p);
    return cudaGetLastError();
  });
}
template <class X, class R, class O>
cudaError_t by_mode(const RmsParams& p, cudaStream_t st) {
  return p.mode == kWide ? go<X, R, O, kWide>(p, st) : p.mode == kShift ? go<X, R, O, kShift>(p, st) : go<X, R, O, kScalar>(p, st);
}
template <class X, class R>
cudaError_t by_out(const RmsParams& p, cudaStream_t st) {
  switch (p.out_type) {
    case kRmsBf16: return by_mode<X, R, bf16>(p, st);
    case kRmsF32: return by_mode<X, R, float>(p, st);
    default: return by_mode<X, R, e4m3_t>(p, st);
  }
}
template <class X>
cudaError_t by_residual(const RmsParams& p, cudaStream_t st) {
  if (p.residual == nullptr) return by_out<X, none_t>(p, st);
  return p.residual_bf16 ? by_out<X, bf16>(p, st) : by_out<X, float>(p, st);
}

template <class X, class R, class G, int MODE>
cudaError_t go_bwd(const RmsBwdParams& p, int blocks, cudaStream_t st) {
  cudaError_t e = by_width<MODE, true>(room_of(MODE, p.d), [&](auto tpr, auto nv) {
    constexpr int TPR = decltype(tpr)::value;
    const size_t smem = TPR == 32 && p.part != nullptr ? 8 * sizeof(float) * static_cast<size_t>(p.d) : 0;
    rms_norm_bwd_kernel<X, R, G, TPR, MODE, decltype(nv)::value><<<blocks, TPR == 32 ? 256 : TPR, smem, st>>>(p);
    return cudaGetLastError();
  });
  if (e != cudaSuccess || p.part == nullptr) return e;
  return launch_column_sum(p.part, blocks, p.d, p.dw, p.dw_bf16, st);
}
template <class X, class R, class G>
cudaError_t bwd_by_mode(const RmsBwdParams& p, int blocks, cudaStream_t st) {
  return p.mode == kWide    ? go_bwd<X, R, G, kWide>(p, blocks, st)
         : p.mode == kShift ? go_bwd<X, R, G, kShift>(p, blocks, st)
                            : go_bwd<X, R, G, kScalar>(p, blocks, st);
}
template <class X, class R>
cudaError_t bwd_by_grad(const RmsBwdParams& p, int blocks, cudaStream_t st) {
  return p.dh_bf16 ? bwd_by_mode<X, R, bf16>(p, blocks, st) : bwd_by_mode<X, R, float>(p, blocks, st);
}
template <class X>
cudaError_t bwd_by_residual(const RmsBwdParams& p, int blocks, cudaStream_t st) {
  if (p.residual == nullptr && p.dr == nullptr) return bwd_by_grad<X, none_t>(p, blocks, st);
  return p.residual_bf16 ? bwd_by_grad<X, bf16>(p, blocks, st) : bwd_by_grad<X, float>(p, blocks, st);
}

}  // namespace

int rms_mode(bool wide, bool packed, int d) { return wide ? kWide : packed && d + 7 <= kRmsMaxWidth ? kShift : kScalar; }

cudaError_t launch_rms_norm(const RmsParams& p, cudaStream_t st) {
  if (p.rows == 0) return cudaSuccess;
  return p.x_bf16 ? by_residual<bf16>(p, st) : by_residual<float>(p, st);
}

// Blocks of the gradient's kernel: as many as are resident, which leaves the most rows to spread the cost of a block's row
// of partials over; a multiple of eight where a block is a row's (mode kShift needs it).
template <int MODE>
int bwd_blocks(int64_t rows, int d, int sms) {
  int blocks = 0;
  by_width<MODE, true>(room_of(MODE, d), [&](auto tpr, auto nv) {
    constexpr int TPR = decltype(tpr)::value;
    const int64_t most = TPR == 32 ? (rows + 7) / 8 : rows;
    const int64_t some = std::min<int64_t>(most, static_cast<int64_t>(sms) * bwd_resident(TPR, decltype(nv)::value * (MODE == kScalar ? 1 : 8)));
    blocks = static_cast<int>(TPR == 32 ? some : (some + 7) / 8 * 8);
    return cudaSuccess;
  });
  return blocks;
}
int rms_bwd_blocks(int64_t rows, int d, int sms, int mode) {
  return mode == kWide ? bwd_blocks<kWide>(rows, d, sms) : mode == kShift ? bwd_blocks<kShift>(rows, d, sms) : bwd_blocks<kScalar>(rows, d, sms);
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
