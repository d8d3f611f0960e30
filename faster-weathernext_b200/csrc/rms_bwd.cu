// Gradient of the root-mean-square norm (rms.cu).
#include "rms_rows.cuh"

namespace fwn {

namespace {

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
}  // namespace fwn
