// Root-mean-square norm of a residual stream, with the residual's addition, an 8-bit output with scales, and its
// gradient:
//   s = x + residual,  rstd = 1 / sqrt(mean(s^2) + eps),  h = s rstd weight
// (x, s float32 or bf16, residual and weight float32, bf16 or absent, h bf16, float32, or e4m3 with one float32 scale
// per row, scale = max |h| / 448, h = scale * value). Sums are float32; s is normalised unrounded and rounded once,
// where it is stored.
//
// Bound: HBM. A row is read once, kept in registers (at most 32 values per thread) through the sum of squares (and the
// row maximum of the 8-bit output) and written once. 8 to 512 threads take a row (the gradient, kShift and kScalar: to
// 1,024, whose 64 registers a thread spill 36 to 368 bytes forward and 460 to 664 in the gradient; its other forms spill
// up to 204), the smallest group that holds it in registers: it needs the fewest exchanges and has the most bytes on their
// way per thread; where those are few (bf16 rows), a group takes up to four rows at once. Three ways to lay a row over its
// threads:
//   kWide    8 values per thread and access (16 bytes of bf16, 32 of float32, the widest accesses of sm_100): widths
//            and strides that are multiples of 8;
//   kShift   the same accesses for rows of any width that follow one another without gaps: groups of 8 start at the
//            aligned address before the row, and only the two that its ends cut go by single values. A group of threads
//            takes rows eight apart, whose starts are off alike, so that a thread keeps its columns (its weights, its
//            share of the weight's gradient) from row to row, and the next row's loads are issued before the work on
//            one. 10,242 x 1,001 bf16 with a bf16 residual, forward / backward: kScalar 41 / 165 us, kShift 19 / 36;
//   kScalar  one value per thread and access: other strides and addresses.
// Measured (of the measured copy rate, 6,468 GB/s): 163,848 x 512, float32 stream + bf16 residual -> bf16 147 us (1.05),
// -> e4m3 136 us (1.05), gradient 225 us (0.93: five arrays of a thread's values keep it to two blocks per SM); 60M
// values of bf16 without a residual 41-47 us at widths of 512 to 4,096 (0.8-0.9: few bytes per row), odd widths 57-97.
// Rows brought to 8 bits alone: 163,848 x 512 of float32 66 us (0.98), of bf16 50 (0.78).
#include "rms_rows.cuh"

namespace fwn {

namespace {

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

}  // namespace

int rms_mode(bool wide, bool packed, int d) { return wide ? kWide : packed && d + 7 <= kRmsMaxWidth ? kShift : kScalar; }

cudaError_t launch_rms_norm(const RmsParams& p, cudaStream_t st) {
  if (p.rows == 0) return cudaSuccess;
  return p.x_bf16 ? by_residual<bf16>(p, st) : by_residual<float>(p, st);
}

cudaError_t launch_column_sum(const float* part, int64_t rows, int d, void* out, bool out_bf16, cudaStream_t st) {
  column_sum_kernel<<<(d + 31) / 32, 1024, 0, st>>>(part, rows, d, out, out_bf16);
  return cudaGetLastError();
}

}  // namespace fwn
