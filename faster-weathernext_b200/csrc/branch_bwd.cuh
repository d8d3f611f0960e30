// Gradient of the residual branch (branch.cu), compiled once for each type of the stream. With yhat = y rstd(y), shat =
// s rstd(s), a = post_weight gate, g = dh weight:
//   dt = rstd(s) (g - shat mean(g shat)) + ds,  dx = alpha dt,  db = dt m,
//   dy = rstd(y) (db a - yhat mean(db a yhat)),
//   d_weight = sum over rows of dh shat,  u = sum over a gate's rows of db yhat,
//   d_gate = post_weight u,  d_post_weight = sum over gates of gate u:
// one sum per column and gate gives both. s and the mask are computed again from x and y and the two saved rstd of a row,
// so that the row's two sums are all that is exchanged, and the written (rounded) s is not read.
//
// Bound: HBM, a row of each tensor read and written once. A group of threads walks rows of one gate after another, the next
// row's loads ahead; its columns' sums stay in registers and leave as one row of partials per block and gate slice, added
// in order by branch_bwd_finish: no atomics, the same bits every time.
#pragma once

#include "branch.cuh"
#include "rms_rows.cuh"

namespace fwn {

namespace {

template <class F>
cudaError_t branch_bwd_width(int room, F f) {
  using std::integral_constant;
#define FWN_ROW(TPR) \
  if (room <= TPR * 8) return f(integral_constant<int, TPR>())
  FWN_ROW(8);
  FWN_ROW(16);
  FWN_ROW(32);
  FWN_ROW(64);
  FWN_ROW(128);
  FWN_ROW(256);
  FWN_ROW(512);
  FWN_ROW(1024);
#undef FWN_ROW
  return cudaErrorInvalidValue;
}
constexpr int branch_bwd_resident(int tpr) { return tpr > 512 ? 1 : 512 / block_of(tpr); }

template <class X, class Y, class G, int TPR, int MODE>
__global__ void __launch_bounds__(block_of(TPR), branch_bwd_resident(TPR)) branch_bwd_kernel(const BranchBwdParams p) {
  constexpr int V = 8, GROUPS = block_of(TPR) / TPR, PER_WARP = TPR < 32 ? 32 / TPR : 1;
  extern __shared__ float part_smem[];  // more than one group: a row of d each
  __shared__ float red[2][1][32];
  const int d = p.d, group = threadIdx.x / TPR;
  const float over = 1.f / static_cast<float>(d);
  const bool drops = p.drop.threshold > 0;
  const uint64_t seed = drops ? drop_seed(p.drop) : 0;
  const int64_t span = p.gates > 1 ? p.gate_span : p.rows, step = static_cast<int64_t>(p.slices) * GROUPS;
  float dw[V], w[V];
#pragma unroll
  for (int e = 0; e < V; ++e) dw[e] = 0.f;
  int off = 0;
  // A block's row of partials: its groups' sums, added in order.
  auto leave = [&](float (&v)[V], float* to) {
    const int j = group_at<TPR, V>(0, off);
    float* mine = GROUPS > 1 ? part_smem + group * d : to;
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (j + e >= 0 && j + e < d) mine[j + e] = v[e];
    if constexpr (GROUPS > 1) {
      __syncthreads();
      for (int c = threadIdx.x; c < d; c += blockDim.x) {
        float t = 0.f;
#pragma unroll 8
        for (int q = 0; q < GROUPS; ++q) t += part_smem[q * d + c];
        to[c] = t;
      }
      __syncthreads();
    }
  };
  for (int item = blockIdx.x; item < p.gates * p.slices; item += gridDim.x) {
    const int gate = item / p.slices, slice = item % p.slices;
    const int64_t end = (gate + 1) * span;
    int64_t row = gate * span + static_cast<int64_t>(slice) * GROUPS + group;
    if (MODE == kShift) off = static_cast<int>(row * d & 7);  // of all the item's rows; a block takes one item
    const int j = group_at<TPR, V>(0, off);
    float a[V], u[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      a[e] = 1.f;
      w[e] = 1.f;
      u[e] = 0.f;
    }
    if (p.post_weight != nullptr) weight_group<MODE>(p.post_weight, p.post_bf16, j, d, a);
    if (p.weight != nullptr) weight_group<MODE>(p.weight, p.weight_bf16, j, d, w);
    if (p.gate != nullptr && !p.gate_values) {
      float q[V];
      const int64_t at = static_cast<int64_t>(gate) * d;
      weight_group<MODE>(p.gate_bf16 ? static_cast<const void*>(static_cast<const bf16*>(p.gate) + at)
                                     : static_cast<const void*>(static_cast<const float*>(p.gate) + at),
                         p.gate_bf16, j, d, q);
#pragma unroll
      for (int e = 0; e < V; ++e) a[e] *= q[e];
    }
    Raw<X, V> nx, nds;
    Raw<Y, V> ny;
    Raw<G, V> ng;
    float2 nr;
    auto fetch = [&](int64_t r) {
      const int n = r < end ? d : 0;
      const bool more = (p.rows - 1 - r) * d >= V - 1;
      nr = n > 0 ? __ldg(reinterpret_cast<const float2*>(p.rstd) + r) : make_float2(0.f, 0.f);
      load_group<MODE>(static_cast<const X*>(p.x) + r * p.x_stride, j, n, more, nx);
      load_group<MODE>(static_cast<const Y*>(p.y) + r * p.y_stride, j, n, more, ny);
      if (p.dh != nullptr) load_group<MODE>(static_cast<const G*>(p.dh) + r * d, j, n, more, ng);
      if (p.ds != nullptr) load_group<MODE>(static_cast<const X*>(p.ds) + r * d, j, n, more, nds);
    };
    fetch(row);
    for (; row - group % PER_WARP < end; row += step) {
      const int n = row < end ? d : 0;
      const float r1 = nr.x, r2 = nr.y;
      float x[V], yh[V], g[V], dt[V], sum[1] = {0.f};
      expand<MODE>(nx, j, n, x);
      expand<MODE>(ny, j, n, yh);
#pragma unroll
      for (int e = 0; e < V; ++e) g[e] = dt[e] = 0.f;
      if (p.dh != nullptr) expand<MODE>(ng, j, n, g);
      if (p.ds != nullptr) expand<MODE>(nds, j, n, dt);
      if (row + step - group % PER_WARP < end) fetch(row + step);
      float gv[V], b[V], m[V];
      if (p.gate_values) {
        const int64_t at = row * d;
        const bool more = (p.rows - 1 - row) * d >= V - 1;
        if (p.gate_bf16) {
          Raw<bf16, V> q;
          load_group<MODE>(static_cast<const bf16*>(p.gate) + at, j, n, more, q);
          expand<MODE>(q, j, n, gv);
        } else {
          Raw<float, V> q;
          load_group<MODE>(static_cast<const float*>(p.gate) + at, j, n, more, q);
          expand<MODE>(q, j, n, gv);
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        yh[e] *= r1;
        b[e] = yh[e] * a[e];
        if (p.gate_values) b[e] *= gv[e];
        m[e] = 1.f;
      }
      if (drops) {
        // The mask's factors, from which b and db both take theirs. A dropped value may be anything: it counts as 0.
        drop8(p.drop, seed, static_cast<uint64_t>(row * d + j) >> 3, m);
#pragma unroll
        for (int e = 0; e < V; ++e) b[e] = m[e] != 0.f ? b[e] * m[e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x[e] = fmaf(p.alpha, x[e], b[e]) * r2;  // shat
        dw[e] = fmaf(g[e], x[e], dw[e]);
        g[e] *= w[e];
        sum[0] = fmaf(g[e], x[e], sum[0]);
      }
      row_reduce<TPR, false>(sum, red[0]);
      const float c1 = sum[0] * over;
      sum[0] = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        dt[e] = fmaf(r2, fmaf(-x[e], c1, g[e]), dt[e]);
        x[e] = p.alpha * dt[e];
      }
      if (p.dx != nullptr) store_group<MODE>(static_cast<X*>(p.dx) + row * d, j, n, x);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        dt[e] = drops ? (m[e] != 0.f ? dt[e] * m[e] : 0.f) : dt[e];  // db
        x[e] = dt[e] * a[e];
        if (p.gate_values) {
          // d_gate = db post_weight yhat (a is post_weight here), and the gate goes into db for the other two.
          b[e] = x[e] * yh[e];
          x[e] *= gv[e];
          dt[e] *= gv[e];
        }
        u[e] = fmaf(dt[e], yh[e], u[e]);
        sum[0] = fmaf(x[e], yh[e], sum[0]);
      }
      if (p.gate_values && p.d_gate != nullptr) {
        if (p.gate_bf16)
          store_group<MODE>(static_cast<bf16*>(p.d_gate) + row * d, j, n, b);
        else
          store_group<MODE>(static_cast<float*>(p.d_gate) + row * d, j, n, b);
      }
      row_reduce<TPR, false>(sum, red[1]);
      const float c2 = sum[0] * over;
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = r1 * fmaf(-yh[e], c2, x[e]);
      if (p.dy != nullptr) store_group<MODE>(static_cast<Y*>(p.dy) + row * d, j, n, x);
    }
    if (p.part_u != nullptr) leave(u, p.part_u + static_cast<int64_t>(item) * d);
  }
  if (p.part_w != nullptr) leave(dw, p.part_w + static_cast<int64_t>(blockIdx.x) * d);
}

template <class X, class Y, class G, int MODE>
cudaError_t go_branch_bwd(const BranchBwdParams& p, cudaStream_t st) {
  return branch_bwd_width(room_of(MODE, p.d), [&](auto tpr) {
    constexpr int TPR = decltype(tpr)::value;
    const size_t smem = block_of(TPR) > TPR ? block_of(TPR) / TPR * sizeof(float) * static_cast<size_t>(p.d) : 0;
    branch_bwd_kernel<X, Y, G, TPR, MODE><<<p.blocks, block_of(TPR), smem, st>>>(p);
    return cudaGetLastError();
  });
}
template <class X, class Y>
cudaError_t branch_bwd_by(const BranchBwdParams& p, cudaStream_t st) {
  if (p.dh_bf16) return p.wide ? go_branch_bwd<X, Y, bf16, kWide>(p, st) : go_branch_bwd<X, Y, bf16, kShift>(p, st);
  return p.wide ? go_branch_bwd<X, Y, float, kWide>(p, st) : go_branch_bwd<X, Y, float, kShift>(p, st);
}

}  // namespace

}  // namespace fwn
