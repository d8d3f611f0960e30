// Root-mean-square norm of a residual stream, with the residual's addition, an 8-bit output with scales, and its
// gradient:
//   s = x + residual,  rstd = 1 / sqrt(mean(s^2) + eps),  h = s rstd weight
// (x, s float32 or bf16, residual and weight float32, bf16 or absent, h bf16, float32, or e4m3 with one float32 scale
// per row, scale = max |h| / 448, h = scale * value). Sums are float32; s is normalised unrounded and rounded once,
// where it is stored.
//
// Bound: HBM. A row is read once, kept in registers (at most 32 values per thread) through the sum of squares (and the
// row maximum of the 8-bit output) and written once. 8 to 512 threads take a row (the gradient: to 1,024), the smallest
// group that holds it in registers: it needs the fewest exchanges and has the most bytes on their way per thread; where
// those are few (bf16 rows), a group takes up to four rows at once. Three ways to lay a row over its threads:
//   kWide    8 values per thread and access (16 bytes of bf16, 32 of float32, the widest accesses of sm_100): widths
//            and strides that are multiples of 8;
//   kShift   the same accesses for rows of any width that follow one another without gaps: groups of 8 start at the
//            aligned address before the row, and only the two that its ends cut go by single values. A group of threads
//            takes rows eight apart, whose starts are off alike, so that a thread keeps its columns (its weights, its
//            share of the weight's gradient) from row to row, and the next row's loads are issued before the work on
//            one. 10,242 x 1,001 bf16 with a bf16 residual, forward / backward: kScalar 41 / 165 us, kShift 19 / 36;
//   kScalar  one value per thread and access: other strides and addresses.
// Measured (of the measured copy rate, 6,468 GB/s): 163,848 x 512, float32 stream + bf16 residual -> bf16 147 us (1.05),
// -> e4m3 135 us (1.05), gradient 224 us (0.93: five arrays of a thread's values keep it to two blocks per SM); 60M
// values of bf16 without a residual 41-47 us at widths of 512 to 4,096 (0.8-0.9: few bytes per row), odd widths 57-97.
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

// Threads of a block whose rows take TPR threads: eight rows or more where a row is at most a warp's, else one.
constexpr int block_of(int tpr) { return tpr <= 32 ? 256 : tpr; }

// Sums (or NaN-keeping maxima) of N values over the TPR threads of a row, the same in each. `red` (N x 32) holds one value
// per warp and is written once per row, so that rows alternate between two of them.
template <int TPR, bool MAX, int N>
__device__ __forceinline__ void row_reduce(float (&v)[N], float (*red)[32]) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float u = __shfl_xor_sync(0xffffffffu, v[i], o);
      v[i] = MAX ? max_nan(v[i], u) : v[i] + u;
    }
  }
  if constexpr (TPR > 32) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((threadIdx.x & 31) == 0) red[i][threadIdx.x >> 5] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = red[i][threadIdx.x & (TPR / 32 - 1)];
#pragma unroll
      for (int o = TPR / 64; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, v[i], o);
        v[i] = MAX ? max_nan(v[i], u) : v[i] + u;
      }
    }
  }
}

enum RowMode { kScalar = 0, kWide = 1, kShift = 2 };

// Column of a thread's i-th group of V values; `off` (kShift) is how far the row starts past an aligned address.
template <int TPR, int V>
__device__ __forceinline__ int group_at(int i, int off) {
  return (i * TPR + static_cast<int>(threadIdx.x & (TPR - 1))) * V - off;
}
// The group of values from column j of the row at p. `more`: V - 1 values or more follow the row, so that a group which
// its end cuts may be read whole (kShift: what lies before a row is the row before); the last rows' go by single values.
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

// The rows of a group of TPR threads: `row`, then `step` further on each time. Groups of one warp have adjacent rows and
// leave together (`base`, the row of the warp's first group, decides); kShift: `step` is a multiple of eight.
template <int TPR>
struct Rows {
  int64_t row, base, step;
  __device__ __forceinline__ Rows() {
    constexpr int GROUPS = block_of(TPR) / TPR, PER_WARP = TPR < 32 ? 32 / TPR : 1;
    const int g = threadIdx.x / TPR;
    row = static_cast<int64_t>(blockIdx.x) * GROUPS + g;
    base = row - g % PER_WARP;
    step = static_cast<int64_t>(gridDim.x) * GROUPS;
  }
};

// Rows that a group works on at once, so that a thread has some 64 bytes on their way: bf16 rows of few values per thread.
template <class X, class R, int MODE>
constexpr int rows_at_once(int nv) {
  if (MODE != kWide) return MODE == kShift && nv == 1 && sizeof(X) == 2 ? 2 : 1;
  const int bytes = nv * 8 * (static_cast<int>(sizeof(X)) + (is_none<R> ? 0 : static_cast<int>(sizeof(R))));
  return bytes <= 16 ? 4 : bytes <= 32 ? 2 : 1;
}

// TPR threads per row, NV groups of V values per thread.
template <class X, class R, class O, int TPR, int MODE, int NV>
__global__ void __launch_bounds__(block_of(TPR), TPR > 512 ? 1 : (MODE == kWide && TPR <= 32 && NV <= 2 ? 1024 : 512) / block_of(TPR))
    rms_norm_kernel(const RmsParams p) {
  constexpr int V = MODE == kScalar ? 1 : 8;
  constexpr int U = rows_at_once<X, R, MODE>(NV);
  __shared__ float red[2][2][U][32];
  Rows<TPR> at;
  const int off = MODE == kShift ? static_cast<int>(at.row * p.d & 7) : 0;  // of all this group's rows
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
  // kShift: the next rows are on their way while some are worked on.
  constexpr bool kAhead = MODE == kShift;
  Raw<X, V> xs[kAhead ? U : 1][kAhead ? NV : 1];
  Raw<RR, V> rs[kAhead ? U : 1][kAhead ? NR : 1];
  auto fetch = [&](int64_t row, int i, Raw<X, V>& a, Raw<RR, V>& b) {
    const int j = group_at<TPR, V>(i, off), n = row < p.rows ? d : 0;
    const bool more = (p.rows - 1 - row) * d >= V - 1;
    load_group<MODE>(static_cast<const X*>(p.x) + row * p.x_stride, j, n, more, a);
    if constexpr (!is_none<R>) load_group<MODE>(static_cast<const R*>(p.residual) + row * p.residual_stride, j, n, more, b);
  };
  auto fetch_rows = [&](int64_t row) {
    if constexpr (kAhead) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < NV; ++i) fetch(row + u * at.step, i, xs[u][i], rs[u][is_none<R> ? 0 : i]);
    }
  };
  fetch_rows(at.row);
  int flip = 0;
  for (; at.base < p.rows; at.base += U * at.step, at.row += U * at.step, flip ^= 1) {
    float s[U][NV][V], ss[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n = at.row + u * at.step < p.rows ? d : 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = group_at<TPR, V>(i, off);
        Raw<X, V> a;
        Raw<RR, V> b;
        if constexpr (kAhead) {
          a = xs[u][i];
          b = rs[u][is_none<R> ? 0 : i];
        } else {
          fetch(at.row + u * at.step, i, a, b);
        }
        expand<MODE>(a, j, n, s[u][i]);
        if constexpr (!is_none<R>) {
          float r[V];
          expand<MODE>(b, j, n, r);
#pragma unroll
          for (int e = 0; e < V; ++e) s[u][i][e] += r[e];
        }
      }
    }
    if constexpr (kAhead) {
      if (at.base + U * at.step < p.rows) fetch_rows(at.row + U * at.step);
    }
    float rstd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = at.row + u * at.step;
      const int n = row < p.rows ? d : 0;
      ss[u] = 0.f;
      rstd[u] = 1.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if constexpr (!is_none<R>) store_group<MODE>(static_cast<X*>(p.x_out) + row * d, group_at<TPR, V>(i, off), n, s[u][i]);
#pragma unroll
        for (int e = 0; e < V; ++e) ss[u] = fmaf(s[u][i][e], s[u][i][e], ss[u]);
      }
    }
    if (p.normalize) {
      row_reduce<TPR, false>(ss, red[flip][0]);
#pragma unroll
      for (int u = 0; u < U; ++u) rstd[u] = rsqrtf(ss[u] / static_cast<float>(d) + p.eps);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (MODE != kShift && p.weight != nullptr)
        weight_group<MODE>(p.weight, p.weight_bf16, group_at<TPR, V>(i, off), d, w[0]);
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          s[u][i][e] *= rstd[u];
          if (MODE == kShift || p.weight != nullptr) s[u][i][e] *= w[MODE == kShift ? i : 0][e];
        }
      }
    }
    if constexpr (sizeof(O) == 1) {
      float m[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        m[u] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < V; ++e) m[u] = max_nan(m[u], fabsf(s[u][i][e]));
      }
      row_reduce<TPR, true>(m, red[flip][1]);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = at.row + u * at.step;
        const bool tiny = m[u] < kTinyRow;  // false for NaN, which the scale and the values keep
        const float inv = tiny ? 0.f : kE4m3Max / m[u];
        if ((threadIdx.x & (TPR - 1)) == 0 && row < p.rows) p.scale[row] = tiny ? 0.f : m[u] / kE4m3Max;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < V; ++e) s[u][i][e] *= inv;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = at.row + u * at.step;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        store_group<MODE>(static_cast<O*>(p.out) + row * d, group_at<TPR, V>(i, off), row < p.rows ? d : 0, s[u][i]);
    }
  }
}

// Blocks of the gradient's kernel that an SM holds: five arrays of a thread's values and some 40 registers a thread, or
// fewer where no row is read ahead.
template <class X, int MODE>
constexpr bool bwd_ahead(int nv) { return nv == 1 && (MODE == kShift || sizeof(X) == 2); }
template <class X, int MODE>
constexpr int bwd_at_once(int nv) { return MODE == kWide && nv == 1 && sizeof(X) == 2 ? 2 : 1; }  // rows, as rows_at_once
template <class X, int MODE>
constexpr int bwd_resident(int tpr, int nv) {
  return tpr > 512 ? 1 : (MODE == kWide && nv == 1 && !bwd_ahead<X, MODE>(nv) ? 768 : 512) / block_of(tpr);
}

// Gradient, with g = dh weight, s the normalised row (x, or x + residual), ds the gradient of the stored sum:
//   dx = rstd g - s rstd^3 mean(g s) + ds,  d_residual = dx,  dweight = sum over rows of dh s rstd.
// A group of TPR threads walks rows; its columns' share of dweight stays in registers and leaves as one row of partials
// per block (a block's groups are added through shared memory), summed in order by column_sum_kernel: no atomics, the
// same bits every time. All of a row's loads are issued before its sums are needed.
template <class X, class R, class G, int TPR, int MODE, int NV>
__global__ void __launch_bounds__(block_of(TPR), (bwd_resident<X, MODE>(TPR, NV)))
    rms_norm_bwd_kernel(const RmsBwdParams p) {
  constexpr int V = MODE == kScalar ? 1 : 8;
  constexpr int GROUPS = block_of(TPR) / TPR;
  extern __shared__ float part_smem[];  // more than one group, with a weight: a row of d each
  constexpr int U = bwd_at_once<X, MODE>(NV);
  __shared__ float red[2][2 * U][32];
  Rows<TPR> at;
  const int off = MODE == kShift ? static_cast<int>(at.row * p.d & 7) : 0;
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
  constexpr bool kAhead = bwd_ahead<X, MODE>(NV);  // the next rows are on their way while some are worked on
  struct Loads {
    Raw<X, V> x, ds;
    Raw<G, V> g;
    Raw<RR, V> r;
  };
  Loads next[U];
  auto fetch = [&](int64_t row, int i, Loads& l) {
    const bool more = (p.rows - 1 - row) * d >= V - 1;
    const int j = group_at<TPR, V>(i, off), n = row < p.rows ? d : 0;
    load_group<MODE>(static_cast<const X*>(p.x) + row * p.x_stride, j, n, more, l.x);
    load_group<MODE>(static_cast<const G*>(p.dh) + row * d, j, n, more, l.g);
    if (p.ds != nullptr) load_group<MODE>(static_cast<const X*>(p.ds) + row * d, j, n, more, l.ds);
    if constexpr (!is_none<R>) {
      if (p.residual != nullptr)
        load_group<MODE>(static_cast<const R*>(p.residual) + row * p.residual_stride, j, n, more, l.r);
    }
  };
  if constexpr (kAhead) {
#pragma unroll
    for (int u = 0; u < U; ++u) fetch(at.row + u * at.step, 0, next[u]);
  }
  int flip = 0;
  for (; at.base < p.rows; at.base += U * at.step, at.row += U * at.step, flip ^= 1) {
    float s[U][NV][V], g[U][NV][V], ds[U][NV][V], sums[2 * U];  // sums: s^2 and g s of each row
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = at.row + u * at.step;
      const int n = row < p.rows ? d : 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = group_at<TPR, V>(i, off);
        Loads l;
        if constexpr (kAhead) l = next[u]; else fetch(row, i, l);
        expand<MODE>(l.x, j, n, s[u][i]);
        expand<MODE>(l.g, j, n, g[u][i]);
        if (p.ds != nullptr) {
          expand<MODE>(l.ds, j, n, ds[u][i]);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) ds[u][i][e] = 0.f;
        }
        if constexpr (!is_none<R>) {
          if (p.residual != nullptr) {
            float r[V];
            expand<MODE>(l.r, j, n, r);
#pragma unroll
            for (int e = 0; e < V; ++e) s[u][i][e] += r[e];
          }
        }
      }
    }
    if constexpr (kAhead) {
      if (at.base + U * at.step < p.rows) {
#pragma unroll
        for (int u = 0; u < U; ++u) fetch(at.row + (U + u) * at.step, 0, next[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      sums[2 * u] = sums[2 * u + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          sums[2 * u] = fmaf(s[u][i][e], s[u][i][e], sums[2 * u]);
          sums[2 * u + 1] = fmaf(g[u][i][e] * w[i][e], s[u][i][e], sums[2 * u + 1]);
        }
      }
    }
    row_reduce<TPR, false>(sums, red[flip]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = at.row + u * at.step;
      const int n = row < p.rows ? d : 0;
      // A row past the end adds nothing (its g and s are 0; with eps = 0 its rstd would be infinite).
      const float rstd = n > 0 ? rsqrtf(sums[2 * u] / static_cast<float>(d) + p.eps) : 0.f;
      const float c = sums[2 * u + 1] / static_cast<float>(d) * rstd * rstd;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = group_at<TPR, V>(i, off);
        float dx[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          dw[i][e] = fmaf(g[u][i][e], s[u][i][e] * rstd, dw[i][e]);
          dx[e] = fmaf(rstd, g[u][i][e] * w[i][e] - s[u][i][e] * c, ds[u][i][e]);
        }
        if (p.dx != nullptr) store_group<MODE>(static_cast<X*>(p.dx) + row * d, j, n, dx);
        if constexpr (!is_none<R>) {
          if (p.dr != nullptr) store_group<MODE>(static_cast<R*>(p.dr) + row * d, j, n, dx);
        }
      }
    }
  }
  if (p.part == nullptr) return;
  float* mine = GROUPS > 1 ? part_smem + threadIdx.x / TPR * d : p.part + static_cast<int64_t>(blockIdx.x) * d;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = group_at<TPR, V>(i, off);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (j + e >= 0 && j + e < d) mine[j + e] = dw[i][e];
  }
  if constexpr (GROUPS > 1) {
    __syncthreads();
    for (int j = threadIdx.x; j < d; j += blockDim.x) {
      float t = 0.f;
#pragma unroll 8
      for (int v = 0; v < GROUPS; ++v) t += part_smem[v * d + j];
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

// Calls f with the threads per row and the groups of values per thread that hold `room` values. The gradient (GRAD,
// which keeps five arrays of a thread's values) and kShift (which reads ahead) take at most two groups, both together one up to 2,048.
template <int MODE, bool GRAD, class F>
cudaError_t by_width(int room, F f) {
  using std::integral_constant;
#define FWN_ROW(TPR, NV) \
  if (room <= TPR * NV * (MODE == kScalar ? 1 : 8)) return f(integral_constant<int, TPR>(), integral_constant<int, NV>())
  if constexpr (MODE == kScalar) {
    FWN_ROW(256, 8);
    FWN_ROW(256, 16);
    FWN_ROW(1024, 16);
  } else {
    FWN_ROW(8, 1);
    FWN_ROW(16, 1);
    FWN_ROW(32, 1);
    if constexpr (MODE != kShift || !GRAD) FWN_ROW(32, 2);
    if constexpr (MODE == kShift && GRAD) {
      FWN_ROW(64, 1);
      FWN_ROW(128, 1);
      FWN_ROW(256, 1);
      FWN_ROW(256, 2);
      FWN_ROW(512, 2);
      FWN_ROW(1024, 2);
    } else if constexpr (GRAD || MODE == kShift) {
      FWN_ROW(64, 2);
      FWN_ROW(128, 2);
      FWN_ROW(256, 2);
      FWN_ROW(512, 2);
      FWN_ROW(1024, 2);
    } else {
      FWN_ROW(32, 3);
      FWN_ROW(32, 4);
      FWN_ROW(64, 3);
      FWN_ROW(64, 4);
      FWN_ROW(128, 3);
      FWN_ROW(128, 4);
      FWN_ROW(256, 4);
      FWN_ROW(512, 4);
    }
  }
#undef FWN_ROW
  return cudaErrorInvalidValue;
}
int room_of(int mode, int d) { return mode == kShift ? d + 7 : d; }

template <class X, class R, class O, int MODE>
cudaError_t go(const RmsParams& p, cudaStream_t st) {
  return by_width<MODE, false>(room_of(MODE, p.d), [&](auto tpr, auto nv) {
    constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, GROUPS = block_of(TPR) / TPR;
    constexpr int U = rows_at_once<X, R, MODE>(NV);
    // kWide, kScalar: the grid covers the rows. kShift: as many blocks as are resident walk them, so that the weights are
    // read once per group of threads; a multiple of eight rows at a step.
    int64_t blocks = (p.rows + GROUPS * U - 1) / (GROUPS * U);
    if (MODE == kShift) {
      blocks = std::min<int64_t>(blocks, static_cast<int64_t>(p.sms) * (TPR > 512 ? 1 : 512 / block_of(TPR)));
      if (GROUPS < 8) blocks = (blocks + 7) / 8 * 8;
    }
    rms_norm_kernel<X, R, O, TPR, MODE, NV><<<static_cast<unsigned>(blocks), block_of(TPR), 0, st>>>(p);
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
    constexpr int GROUPS = block_of(TPR) / TPR;
    const size_t smem = GROUPS > 1 && p.part != nullptr ? GROUPS * sizeof(float) * static_cast<size_t>(p.d) : 0;
    rms_norm_bwd_kernel<X, R, G, TPR, MODE, decltype(nv)::value><<<blocks, block_of(TPR), smem, st>>>(p);
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
template <class X, int MODE>
int bwd_blocks(int64_t rows, int d, int sms) {
  int blocks = 0;
  by_width<MODE, true>(room_of(MODE, d), [&](auto tpr, auto nv) {
    constexpr int TPR = decltype(tpr)::value, GROUPS = block_of(TPR) / TPR;
    const int64_t most = (rows + GROUPS - 1) / GROUPS;
    const int64_t some = std::min<int64_t>(most, static_cast<int64_t>(sms) * bwd_resident<X, MODE>(TPR, decltype(nv)::value));
    blocks = static_cast<int>(GROUPS >= 8 ? some : (some + 7) / 8 * 8);
    return cudaSuccess;
  });
  return blocks;
}
template <class X>
int bwd_blocks_of(int64_t rows, int d, int sms, int mode) {
  return mode == kWide    ? bwd_blocks<X, kWide>(rows, d, sms)
         : mode == kShift ? bwd_blocks<X, kShift>(rows, d, sms)
                          : bwd_blocks<X, kScalar>(rows, d, sms);
}
int rms_bwd_blocks(int64_t rows, int d, int sms, int mode, bool x_bf16) {
  return x_bf16 ? bwd_blocks_of<bf16>(rows, d, sms, mode) : bwd_blocks_of<float>(rows, d, sms, mode);
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
