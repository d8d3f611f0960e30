// What the branch's kernels (branch.cu) and their gradients' (branch_bwd.cuh) share: eight values of a row in packed pairs.
#pragma once

#include "branch.cuh"
#include "packed.cuh"
#include "rms_rows.cuh"

namespace fwn {

namespace {

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

// The values of a group as loaded; columns outside [0, d) are 0.
template <int MODE, class T>
__device__ __forceinline__ V8 values(const Raw<T, 8>& r, int j, int d) {
  V8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = raw_at(r, e);
    set8(v, e, MODE != kShift || (j + e >= 0 && j + e < d) ? x : 0.f);
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
