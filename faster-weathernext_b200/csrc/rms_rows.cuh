// What the RMS norm's kernels (rms.cu) and their gradient's (rms_bwd.cu) share: rows in registers, their accesses in the
// three modes that rms.cu describes, sums over a row's threads, and the choice of threads per row.
#pragma once

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

}  // namespace

}  // namespace fwn
