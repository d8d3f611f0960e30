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
// acc += a b, the even columns' sum and the odd ones'.
__device__ __forceinline__ void dot(float2& acc, const V8& a, const V8& b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = ffma2(a.p[i], b.p[i], acc);
}

// Which of a group's eight columns lie in [0, d), for kShift, where the groups at a row's ends are cut: bits, and masks of the
// words of two bf16 values.
template <int MODE>
struct Cut {
  uint32_t bits, words[MODE == kShift ? 4 : 1];
  Cut() = default;
  __device__ __forceinline__ Cut(int j, int d) : bits(j < d ? 0xFFu : 0u) {
    if constexpr (MODE == kShift) {
      if (j < 0) bits = 0xFFu << -j & 0xFFu;
      if (j < d && j + 8 > d) bits &= (1u << (d - j)) - 1u;
#pragma unroll
      for (int i = 0; i < 4; ++i) words[i] = (bits >> (2 * i) & 1u ? 0xFFFFu : 0u) | (bits >> (2 * i + 1) & 1u ? 0xFFFF0000u : 0u);
    }
  }
};
// The values of a group as loaded; columns that are cut off, which may hold anything, are 0.
template <int MODE>
__device__ __forceinline__ V8 values(const Raw<bf16, 8>& r, const Cut<MODE>& cut) {
  Raw<bf16, 8> m = r;
  if constexpr (MODE == kShift) {
#pragma unroll
    for (int i = 0; i < 4; ++i) m.u[i] &= cut.words[i];
  }
  V8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) set8(v, e, raw_at(m, e));
  return v;
}
template <int MODE>
__device__ __forceinline__ V8 values(const Raw<float, 8>& r, const Cut<MODE>& cut) {
  V8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) set8(v, e, raw_at(r, e));
  if constexpr (MODE == kShift) {
    if (cut.bits != 0xFFu) {
#pragma unroll
      for (int e = 0; e < 8; ++e) set8(v, e, cut.bits >> e & 1u ? at8(v, e) : 0.f);
    }
  }
  return v;
}
// The group from column j of the row of n values at p (0: a row that is not there): a wide access, and single values only at
// the tensor's end, where it would reach past it (not `whole`). What is not loaded is 0. (With the groups past a row's end in
// the single values' loop too, and every column masked by comparisons, 163,848 x 250 bf16 took 132 us forward and 270
// backward.)
template <int MODE, class T>
__device__ __forceinline__ void grab(const T* p, int j, int n, bool whole, Raw<T, 8>& r) {
  if constexpr (MODE == kWide) {
    load_group<MODE>(p, j, n, true, r);
  } else {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(r.u) / 4); ++i) r.u[i] = 0;
    const bool in = n > 0 && j < n, wide = whole || j + 8 <= n;  // j may be below 0: a group that begins in the row before
    if (in && wide) load_raw(p + j, r);
    if (in && !wide) load_group<MODE>(p, j, n, false, r);
  }
}
// The same of kShift, of a row of d values that is `there` or not: one condition for all of a row's tensors. The gradient,
// which reads four, takes this one (40,962 x 1,001 bf16 123 us, with grab 147; 163,848 x 333 244 and 288), the forward the
// other (73, and 78 with this one).
template <class T>
__device__ __forceinline__ void grab_shifted(const T* p, int j, int d, bool there, bool whole, Raw<T, 8>& r) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(r.u) / 4); ++i) r.u[i] = 0;
  const bool quick = there && whole;
  if (quick && j < d) load_raw(p + j, r);
  if (there && !quick && j < d) load_group<kShift>(p, j, d, false, r);
}
// Rows before this one are followed by seven values or more.
__device__ __forceinline__ int64_t whole_rows(int64_t rows, int d) { return rows - (d + 6) / d; }
// Groups that kShift's rows of d values take, in values: a row starts up to 8 - gcd(d, 8) values past an aligned address.
inline int branch_room(int mode, int d) { return mode == kShift ? d + 8 - std::min(8, d & -d) : d; }

// A cut group at p + j: the columns from `lo` on (its row's first), or those before `hi` (its last), in at most three stores
// of one, two and four values, each aligned as the whole is (163,848 x 250 bf16 139 -> 132 us forward, 283 -> 270 backward
// against up to eight stores of one).
__device__ __forceinline__ uint32_t pick(const uint32_t (&w)[4], int i) { return i & 2 ? (i & 1 ? w[3] : w[2]) : (i & 1 ? w[1] : w[0]); }
__device__ __forceinline__ void put_cut(float* p, const V8& v, int lo, int hi) {
  if (lo > 0) {
    if (lo & 1) p[lo] = lo & 4 ? (lo & 2 ? v.p[3].y : v.p[2].y) : (lo & 2 ? v.p[1].y : v.p[0].y);
    const int q = (lo + 1) & ~1;
    if (q & 2) *reinterpret_cast<float2*>(p + q) = q & 4 ? v.p[3] : v.p[1];
    if (lo <= 4) *reinterpret_cast<float4*>(p + 4) = make_float4(v.p[2].x, v.p[2].y, v.p[3].x, v.p[3].y);
  } else {
    if (hi & 4) *reinterpret_cast<float4*>(p) = make_float4(v.p[0].x, v.p[0].y, v.p[1].x, v.p[1].y);
    if (hi & 2) *reinterpret_cast<float2*>(p + (hi & 4)) = hi & 4 ? v.p[2] : v.p[0];
    if (hi & 1) p[hi - 1] = hi & 4 ? (hi & 2 ? v.p[3].x : v.p[2].x) : (hi & 2 ? v.p[1].x : v.p[0].x);
  }
}
__device__ __forceinline__ uint32_t pack2(float2 v) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void put_cut(bf16* out, const V8& v, int lo, int hi) {
  const uint32_t w[4] = {pack2(v.p[0]), pack2(v.p[1]), pack2(v.p[2]), pack2(v.p[3])};
  uint16_t* p = reinterpret_cast<uint16_t*>(out);
  if (lo > 0) {
    if (lo & 1) p[lo] = static_cast<uint16_t>(pick(w, lo >> 1) >> 16);
    const int q = (lo + 1) & ~1;
    if (q & 2) *reinterpret_cast<uint32_t*>(p + q) = q & 4 ? w[3] : w[1];
    if (lo <= 4) *reinterpret_cast<uint2*>(p + 4) = make_uint2(w[2], w[3]);
  } else {
    if (hi & 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    if (hi & 2) *reinterpret_cast<uint32_t*>(p + (hi & 4)) = hi & 4 ? w[2] : w[0];
    if (hi & 1) p[hi - 1] = static_cast<uint16_t>(pick(w, hi >> 1));
  }
}
__device__ __forceinline__ void put_cut(e4m3_t* out, const V8& v, int lo, int hi) {
  const uint32_t w[4] = {pack_e4m3x2(v.p[0].x, v.p[0].y), pack_e4m3x2(v.p[1].x, v.p[1].y), pack_e4m3x2(v.p[2].x, v.p[2].y),
                         pack_e4m3x2(v.p[3].x, v.p[3].y)};
  uint8_t* p = reinterpret_cast<uint8_t*>(out);
  if (lo > 0) {
    if (lo & 1) p[lo] = static_cast<uint8_t>(pick(w, lo >> 1) >> 8);
    const int q = (lo + 1) & ~1;
    if (q & 2) *reinterpret_cast<uint16_t*>(p + q) = static_cast<uint16_t>(q & 4 ? w[3] : w[1]);
    if (lo <= 4) *reinterpret_cast<uint32_t*>(p + 4) = w[2] | w[3] << 16;
  } else {
    if (hi & 4) *reinterpret_cast<uint32_t*>(p) = w[0] | w[1] << 16;
    if (hi & 2) *reinterpret_cast<uint16_t*>(p + (hi & 4)) = static_cast<uint16_t>(hi & 4 ? w[2] : w[0]);
    if (hi & 1) p[hi - 1] = static_cast<uint8_t>(pick(w, hi >> 1));
  }
}
// Eight values to column j of a row of n columns (0: nothing).
template <int MODE, class T>
__device__ __forceinline__ void put(T* p, int j, int n, const V8& v) {
  const float t[8] = {v.p[0].x, v.p[0].y, v.p[1].x, v.p[1].y, v.p[2].x, v.p[2].y, v.p[3].x, v.p[3].y};
  if constexpr (MODE == kShift) {
    if (j >= 0 && j + 8 <= n) {
      store_vals(p + j, t);
    } else if (j < n) {
      if (j >= 0 || j + 8 <= n) {
        put_cut(p + j, v, j < 0 ? -j : 0, n - j);
      } else {  // a row within one group
        store_group<MODE>(p, j, n, t);
      }
    }
  } else {
    store_group<MODE>(p, j, n, t);
  }
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
__device__ __forceinline__ V8 gate_values(const void* gate, bool gate_bf16, int64_t row, int j, int d, bool there, bool whole,
                                          const Cut<MODE>& cut) {
  if (gate_bf16) {
    Raw<bf16, 8> r;
    grab<MODE>(static_cast<const bf16*>(gate) + row * d, j, there ? d : 0, whole, r);
    return values(r, cut);
  }
  Raw<float, 8> r;
  grab<MODE>(static_cast<const float*>(gate) + row * d, j, there ? d : 0, whole, r);
  return values(r, cut);
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
