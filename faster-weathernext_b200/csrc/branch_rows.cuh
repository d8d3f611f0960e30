// What the branch's kernels (branch.cu) and their gradients' (branch_bwd.cuh) share: eight values of a row in packed pairs.
#pragma once

#include "branch.cuh"
#include "packed.cuh"
#include "rms_rows.cuh"

namespace fwn {

namespace {

// How a row lies over threads. TPR > 0: a power of two of a warp's threads, several rows a block of 256. TPR = 0: the whole
// block, of as many warps as the row needs (MAXT at most), so that few threads idle at any width.
template <int TPR>
__device__ __forceinline__ int column_of(int i, int off) {
  return (TPR > 0 ? i * TPR + static_cast<int>(threadIdx.x & (TPR - 1)) : i * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * 8 - off;
}
template <int TPR>
constexpr int groups_of() { return TPR > 0 ? 256 / TPR : 1; }
template <int TPR>
constexpr int per_warp() { return TPR > 0 && TPR < 32 ? 32 / TPR : 1; }
template <int TPR>
__device__ __forceinline__ bool row_first() { return TPR > 0 ? (threadIdx.x & (TPR - 1)) == 0 : threadIdx.x == 0; }

// The sum (or NaN-keeping maximum, of values that are not negative) over a row's threads, the same in each. `red`: 32 zeros
// at first, one value per warp, read back whole; a reduction's red is free again after the next one's barrier.
template <int TPR, bool MAX>
__device__ __forceinline__ float over_row(float v, float* red) {
#pragma unroll
  for (int o = (TPR > 0 ? TPR : 32) / 2; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? max_nan(v, u) : v + u;
  }
  if constexpr (TPR == 0) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float4 t = reinterpret_cast<const float4*>(red)[0];
    for (int w = 4; w < static_cast<int>(blockDim.x >> 5); w += 4) {
      const float4 u = reinterpret_cast<const float4*>(red)[w >> 2];
      t = MAX ? make_float4(max_nan(t.x, u.x), max_nan(t.y, u.y), max_nan(t.z, u.z), max_nan(t.w, u.w))
              : make_float4(t.x + u.x, t.y + u.y, t.z + u.z, t.w + u.w);
    }
    v = MAX ? max_nan(max_nan(t.x, t.y), max_nan(t.z, t.w)) : (t.x + t.y) + (t.z + t.w);
  }
  return v;
}
template <int TPR, int N>
__device__ __forceinline__ void clear_red(float (&red)[N][32]) {
  if constexpr (TPR == 0) {
    for (int i = threadIdx.x; i < N * 32; i += blockDim.x) red[i / 32][i % 32] = 0.f;
    __syncthreads();
  }
}

struct V8 {
  float2 p[4];
};
__device__ __forceinline__ V8 all8(float v) { return {{make_float2(v, v), make_float2(v, v), make_float2(v, v), make_float2(v, v)}}; }
__device__ __forceinline__ float at8(const V8& v, int e) { return e & 1 ? v.p[e / 2].y : v.p[e / 2].x; }
__device__ __forceinline__ void set8(V8& v, int e, float x) { (e & 1 ? v.p[e / 2].y : v.p[e / 2].x) = x; }
__device__ __forceinline__ V8 mul(const V8& a, const V8& b) {
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = fmul2(a.p[i], b.p[i]);
  return r;
}
__device__ __forceinline__ V8 mul(const V8& a, float b) {
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = fmul2(a.p[i], make_float2(b, b));
  return r;
}
__device__ __forceinline__ V8 fma(const V8& a, const V8& b, const V8& c) {
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = ffma2(a.p[i], b.p[i], c.p[i]);
  return r;
}
__device__ __forceinline__ V8 fma(const V8& a, float b, const V8& c) {
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.p[i] = ffma2(a.p[i], make_float2(b, b), c.p[i]);
  return r;
}
// acc += a b, four sums of each half; the whole by sum2.
__device__ __forceinline__ void dot(float2& acc, const V8& a, const V8& b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = ffma2(a.p[i], b.p[i], acc);
}

// The values of a group as loaded; columns outside [0, d), which a group at the row's ends brings, are 0.
template <int MODE, class T>
__device__ __forceinline__ V8 values(const Raw<T, 8>& r, int j, int d) {
  V8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) set8(v, e, raw_at(r, e));
  if constexpr (MODE == kShift) {
    if (j < 0 || j + 8 > d) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (j + e < 0 || j + e >= d) set8(v, e, 0.f);
    }
  }
  return v;
}
template <int MODE, class T>
__device__ __forceinline__ void put(T* p, int j, int d, const V8& v) {
  const float t[8] = {v.p[0].x, v.p[0].y, v.p[1].x, v.p[1].y, v.p[2].x, v.p[2].y, v.p[3].x, v.p[3].y};
  store_group<MODE>(p, j, d, t);
}
// Eight of a row of columns (weights, a gate's row); ones where there is none, 0 outside [0, d).
template <int MODE>
__device__ __forceinline__ V8 columns(const void* w, bool w_bf16, int j, int d) {
  if (w == nullptr) return all8(1.f);
  float t[8];
  weight_group<MODE>(w, w_bf16, j, d, t);
  return {{make_float2(t[0], t[1]), make_float2(t[2], t[3]), make_float2(t[4], t[5]), make_float2(t[6], t[7])}};
}
__device__ __forceinline__ const void* gate_row(const void* gate, bool gate_bf16, int64_t row, int d) {
  return static_cast<const uint8_t*>(gate) + row * d * (gate_bf16 ? 2 : 4);
}
// Eight of a row of a gate that has one for every row: aligned as the row itself is.
template <int MODE>
__device__ __forceinline__ V8 gate_values(const void* gate, bool gate_bf16, int64_t row, int j, int d, int width, bool more) {
  if (gate_bf16) {
    Raw<bf16, 8> r;
    load_group<MODE>(static_cast<const bf16*>(gate) + row * width, j, d, more, r);
    return values<MODE>(r, j, d);
  }
  Raw<float, 8> r;
  load_group<MODE>(static_cast<const float*>(gate) + row * width, j, d, more, r);
  return values<MODE>(r, j, d);
}
// Values that dropout takes become 0, whatever they were.
__device__ __forceinline__ V8 kept(const V8& v, const uint4& words, uint32_t least) {
  V8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) set8(r, e, drop_keeps(words, least, e) ? at8(v, e) : 0.f);
  return r;
}

}  // namespace

}  // namespace fwn
