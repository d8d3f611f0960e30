// A residual branch in one pass: the norm after a block, its gate, dropout, the addition to the scaled residual stream and
// the norm before the next block,
//   z = y rstd(y) post_weight,  s = alpha x + gate z m,  h = s rstd(s) weight,  rstd(v) = 1 / sqrt(mean(v^2) + eps),
// with m dropout's mask (philox.cuh), and dropout alone. x, s float32 or bf16, y, gate and weights float32 or bf16, h bf16,
// float32, or e4m3 with one float32 scale per row (max |h| / 448). Sums are float32, s is normalised unrounded.
//
// Bound: HBM. The two norms need two sums over a row, the second of values that depend on the first: a row stays in
// registers through both, read once and written once. The threads of a row, their accesses (kWide: 8 values an access;
// kShift: the same for contiguous rows of any width, from the aligned address before the row) are the RMS norm's
// (rms_rows.cuh). Resident blocks walk the rows, the next one's loads ahead of the work on one, the columns' factors in
// registers. Measured at 163,848 x 512, float32 stream, bf16 branch (of the measured copy rate): 164 us (0.94), with dropout
// 169 (0.91; bf16 stream 123, 0.83: 110 integer instructions per eight values); 40,962 x 2,048 155 (0.99); 163,848 x 333 138
// (0.72).
#include "branch_rows.cuh"

namespace fwn {

namespace {

// Threads of a row, groups of eight values a thread, and the block's most threads: up to 768 values a warp or less (16 or 24
// values a thread, some 100 bytes on their way), above them a block of as many warps as the row needs (20,481 x 4,096 at eight
// values a thread, one block of 16 warps an SM: 202 us, at sixteen 159). From 513 to 768 values, at 24 a thread and eight warps
// an SM, both come close: 40,962 x 576 bf16 45 us, as blocks of three warps 42, with dropout 53 and 55; float32 stream 55 and 52,
// with dropout 57 and 56; 768 bf16 52 and 48; 761 bf16 63 and 56.
template <class F>
cudaError_t branch_width(int room, F f) {
  using std::integral_constant;
#define FWN_ROW(TPR, NV, MAXT) \
  if (room <= (TPR > 0 ? TPR : MAXT) * NV * 8) return f(integral_constant<int, TPR>(), integral_constant<int, NV>(), integral_constant<int, MAXT>())
  FWN_ROW(8, 1, 256);
  FWN_ROW(8, 2, 256);
  FWN_ROW(8, 3, 256);
  FWN_ROW(16, 2, 256);
  FWN_ROW(16, 3, 256);
  FWN_ROW(32, 2, 256);
  FWN_ROW(32, 3, 256);
  FWN_ROW(0, 1, 128);
  FWN_ROW(0, 1, 256);
  FWN_ROW(0, 2, 256);
  FWN_ROW(0, 2, 512);
#undef FWN_ROW
  return cudaErrorInvalidValue;
}
// Threads of an SM: 255 registers a thread at 24 values, 80 at 8 values of a block's rows, 128 elsewhere.
constexpr int branch_resident(int tpr, int nv) { return nv == 3 ? 256 : tpr == 0 && nv == 1 ? 768 : 512; }

template <class X, class Y, int TPR, int MODE, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT, (branch_resident(TPR, NV) / MAXT)) branch_norm_kernel(const BranchParams p) {
  __shared__ __align__(16) float red[3][32];
  clear_red<TPR>(red);
  // Groups of one warp have adjacent rows and leave together (`base`, the row of the warp's first group, decides).
  struct {
    int64_t row, base, step;
  } at;
  const int group = TPR > 0 ? threadIdx.x / (TPR > 0 ? TPR : 1) : 0;
  at.row = static_cast<int64_t>(blockIdx.x) * groups_of<TPR>() + group;
  at.base = at.row - group % per_warp<TPR>();
  at.step = static_cast<int64_t>(gridDim.x) * groups_of<TPR>();
  const int off = MODE == kShift ? static_cast<int>(at.row * p.d & 7) : 0;  // of all this group's rows
  const int d = p.d;
  const float over = 1.f / static_cast<float>(d);
  const bool one_gate = p.gate == nullptr || p.gate_span >= p.rows, own_gate = p.gate_span == 1 && !one_gate;
  const bool drops = p.drop.threshold > 0;
  const uint32_t least = drop_least(p.drop);
  const float factor = drops ? p.drop.factor : 1.f;
  // The next row is on its way while one is worked on; the columns' factors stay in registers.
  Raw<X, 8> xr[NV];
  Raw<Y, 8> yr[NV];
  const int64_t whole = whole_rows(p.rows, d);
  auto fetch = [&](int64_t row) {
    const int n = row < p.rows ? d : 0;
    const X* x = static_cast<const X*>(p.x) + row * p.x_stride;
    const Y* y = static_cast<const Y*>(p.y) + row * p.y_stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = column_of<TPR>(i, off);
      grab<MODE>(y, j, n, row < whole, yr[i]);
      grab<MODE>(x, j, n, row < whole, xr[i]);
    }
  };
  fetch(at.row);
  Cut<MODE> cut[NV] = {};
#pragma unroll
  for (int i = 0; i < NV; ++i) cut[i] = Cut<MODE>(column_of<TPR>(i, off), d);
  V8 g[NV], w[NV];  // post_weight gate factor, weight
  auto columns_of = [&](int64_t gate) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = column_of<TPR>(i, off);
      g[i] = mul(columns<MODE>(p.post_weight, p.post_bf16, j, d), factor);
      if (p.gate != nullptr && !own_gate) g[i] = mul(g[i], columns<MODE>(gate_row(p.gate, p.gate_bf16, gate, d), p.gate_bf16, j, d));
    }
  };
  int gate = -1;
#pragma unroll
  for (int i = 0; i < NV; ++i) w[i] = columns<MODE>(p.weight, p.weight_bf16, column_of<TPR>(i, off), d);
  if (one_gate || own_gate) columns_of(0);
  const uint64_t seed = drops ? drop_seed(p.drop) : 0;
  for (; at.base < p.rows; at.base += at.step, at.row += at.step) {
    const int64_t row = at.row;
    const int n = row < p.rows ? d : 0;
    if (!one_gate && !own_gate && n > 0) {
      const int mine = static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(p.gate_span));
      if (mine != gate) columns_of(gate = mine);
    }
    V8 s[NV], x[NV];
    float2 acc = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      s[i] = values(yr[i], cut[i]);
      x[i] = mul(values(xr[i], cut[i]), p.alpha);
      dot(acc, s[i], s[i]);
    }
    if (at.base + at.step < p.rows) fetch(row + at.step);
    const float r1 = rsqrtf(over_row<TPR, false>(acc.x + acc.y, red[0]) * over + p.eps);
    acc = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = column_of<TPR>(i, off);
      s[i] = mul(mul(s[i], r1), g[i]);
      if (own_gate) s[i] = mul(s[i], gate_values<MODE>(p.gate, p.gate_bf16, row, j, d, n > 0, row < whole, cut[i]));
      if (drops) s[i] = kept(s[i], drop_words(p.drop, seed, static_cast<uint64_t>(row * d + j) >> 3), least);
#pragma unroll
      for (int q = 0; q < 4; ++q) s[i].p[q] = fadd2(s[i].p[q], x[i].p[q]);
      put<MODE>(static_cast<X*>(p.s) + row * d, j, n, s[i]);
      dot(acc, s[i], s[i]);
    }
    const float r2 = rsqrtf(over_row<TPR, false>(acc.x + acc.y, red[1]) * over + p.eps);
    if (p.rstd != nullptr && row_first<TPR>() && n > 0)
      reinterpret_cast<float2*>(p.rstd)[row] = make_float2(r1, r2);
#pragma unroll
    for (int i = 0; i < NV; ++i) s[i] = mul(mul(s[i], r2), w[i]);
    if (p.out_type == kRmsE4m3) {
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) most = max_nan(most, fabsf(at8(s[i], e)));
      most = over_row<TPR, true>(most, red[2]);
      const bool tiny = most < kTinyRow;  // false for NaN, which the scale and the values keep
      const float inv = tiny ? 0.f : kE4m3Max / most;
      if (row_first<TPR>() && n > 0) p.scale[row] = tiny ? 0.f : most / kE4m3Max;
#pragma unroll
      for (int i = 0; i < NV; ++i) put<MODE>(static_cast<e4m3_t*>(p.h) + row * d, column_of<TPR>(i, off), n, mul(s[i], inv));
    } else if (p.out_type == kRmsBf16) {
#pragma unroll
      for (int i = 0; i < NV; ++i) put<MODE>(static_cast<bf16*>(p.h) + row * d, column_of<TPR>(i, off), n, s[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) put<MODE>(static_cast<float*>(p.h) + row * d, column_of<TPR>(i, off), n, s[i]);
    }
  }
}

template <class X, class Y, int MODE>
cudaError_t go(const BranchParams& p, cudaStream_t st) {
  const int room = branch_room(MODE, p.d);
  return branch_width(room, [&](auto tpr, auto nv, auto maxt) {
    constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, MAXT = decltype(maxt)::value, GROUPS = groups_of<TPR>();
    const int threads = TPR > 0 ? MAXT : (room + 256 * NV - 1) / (256 * NV) * 32;
    // Resident blocks walk the rows (kShift: a multiple of eight rows at a step).
    const int64_t resident = static_cast<int64_t>(p.sms) * (branch_resident(TPR, NV) / threads);
    int64_t blocks = std::min<int64_t>((p.rows + GROUPS - 1) / GROUPS, resident);
    if (MODE == kShift && GROUPS < 8) blocks = (blocks + 7) / 8 * 8;
    branch_norm_kernel<X, Y, TPR, MODE, NV, MAXT><<<static_cast<unsigned>(blocks), threads, 0, st>>>(p);
    return cudaGetLastError();
  });
}
template <class X, class Y>
cudaError_t by_mode(const BranchParams& p, cudaStream_t st) {
  return p.wide ? go<X, Y, kWide>(p, st) : go<X, Y, kShift>(p, st);
}

// ---- dropout alone -------------------------------------------------------------------------------------------------

// U groups of eight values a thread: their loads are on their way together, and they share the generator's keys.
constexpr int kDropGroups = 4;
template <class T, bool WIDE>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, T* __restrict__ out, int64_t n, const DropParams drop) {
  constexpr int U = kDropGroups;
  const uint64_t seed = drop_seed(drop);
  const uint32_t least = drop_least(drop);
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * 256 * U + threadIdx.x;
  Raw<T, 8> r[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t at = (i0 + u * 256) * 8;
    if (WIDE && at + 8 <= n) {
      load_raw(x + at, r[u]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        Raw<T, 1> one;
        one.u[0] = 0;
        if (at + e < n) load_raw(x + at + e, one);
        if constexpr (sizeof(T) == 4)
          r[u].u[e] = one.u[0];
        else
          r[u].u[e / 2] = e & 1 ? r[u].u[e / 2] | one.u[0] << 16 : one.u[0];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t at = (i0 + u * 256) * 8;
    const uint4 words = drop_words(drop, seed, static_cast<uint64_t>(at) >> 3);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = drop_keeps(words, least, e) ? raw_at(r[u], e) * drop.factor : 0.f;
    if (WIDE && at + 8 <= n) {
      store_vals(out + at, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float one[1] = {v[e]};
        if (at + e < n) store_vals(out + at + e, one);
      }
    }
  }
}

template <class T>
cudaError_t dropout_by(const void* x, void* out, int64_t n, bool wide, const DropParams& drop, cudaStream_t st) {
  const int64_t blocks = (n + 256 * 8 * kDropGroups - 1) / (256 * 8 * kDropGroups);
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  if (wide)
    dropout_kernel<T, true><<<static_cast<unsigned>(blocks), 256, 0, st>>>(static_cast<const T*>(x), static_cast<T*>(out), n, drop);
  else
    dropout_kernel<T, false><<<static_cast<unsigned>(blocks), 256, 0, st>>>(static_cast<const T*>(x), static_cast<T*>(out), n, drop);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_branch(const BranchParams& p, cudaStream_t st) {
  if (p.rows == 0) return cudaSuccess;
  if (p.x_bf16) return p.y_bf16 ? by_mode<bf16, bf16>(p, st) : by_mode<bf16, float>(p, st);
  return p.y_bf16 ? by_mode<float, bf16>(p, st) : by_mode<float, float>(p, st);
}

cudaError_t launch_dropout(const void* x, void* out, int64_t n, bool bf16_values, bool wide, const DropParams& drop,
                           cudaStream_t st) {
  if (n == 0) return cudaSuccess;
  return bf16_values ? dropout_by<bf16>(x, out, n, wide, drop, st) : dropout_by<float>(x, out, n, wide, drop, st);
}

}  // namespace fwn
