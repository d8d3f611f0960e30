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

#include "branch_rows.cuh"

namespace fwn {

namespace {

// Threads of a row and groups of eight values a thread.
template <class F>
cudaError_t branch_bwd_width(int room, F f) {
  using std::integral_constant;
#define FWN_ROW(TPR, NV) \
  if (room <= TPR * NV * 8) return f(integral_constant<int, TPR>(), integral_constant<int, NV>())
  FWN_ROW(8, 1);
  FWN_ROW(16, 1);
  FWN_ROW(32, 1);
  FWN_ROW(64, 1);
  FWN_ROW(128, 1);
  FWN_ROW(256, 1);
  FWN_ROW(512, 1);
  FWN_ROW(1024, 1);
#undef FWN_ROW
  return cudaErrorInvalidValue;
}
constexpr int branch_bwd_resident(int tpr, int nv) { return tpr > 512 ? 1 : (nv > 1 ? 256 : 512) / block_of(tpr); }

template <class X, class Y, class G, int TPR, int NV, int MODE>
__global__ void __launch_bounds__(block_of(TPR), (branch_bwd_resident(TPR, NV))) branch_bwd_kernel(const BranchBwdParams p) {
  constexpr int GROUPS = block_of(TPR) / TPR, PER_WARP = TPR < 32 ? 32 / TPR : 1;
  extern __shared__ float part_smem[];  // more than one group: a row of d each
  __shared__ float red[2][1][32];
  const int d = p.d, group = threadIdx.x / TPR;
  const float over = 1.f / static_cast<float>(d);
  const bool drops = p.drop.threshold > 0, own_gate = p.gate_values;
  const uint32_t least = drop_least(p.drop);
  const float factor = drops ? p.drop.factor : 1.f;
  const uint64_t seed = drops ? drop_seed(p.drop) : 0;
  const int64_t span = p.gates > 1 ? p.gate_span : p.rows, step = static_cast<int64_t>(p.slices) * GROUPS;
  V8 dw[NV], w[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) dw[i] = all8(0.f);
  int off = 0;
  // A block's row of partials: its groups' sums, added in order.
  auto leave = [&](const V8 (&v)[NV], float scale, float* to) {
    float* mine = GROUPS > 1 ? part_smem + group * d : to;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = group_at<TPR, 8>(i, off);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (j + e >= 0 && j + e < d) mine[j + e] = at8(v[i], e) * scale;
    }
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
    V8 a[NV], u[NV];  // post_weight gate factor, sums of db yhat (without the factor)
    Raw<X, 8> nx[NV], nds[NV];
    Raw<Y, 8> ny[NV];
    Raw<G, 8> ng[NV];
    float2 nr;
    auto fetch = [&](int64_t r) {
      const int n = r < end ? d : 0;
      const bool more = (p.rows - 1 - r) * d >= 7;
      nr = n > 0 ? __ldg(reinterpret_cast<const float2*>(p.rstd) + r) : make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = group_at<TPR, 8>(i, off);
        load_group<MODE>(static_cast<const X*>(p.x) + r * p.x_stride, j, n, more, nx[i]);
        load_group<MODE>(static_cast<const Y*>(p.y) + r * p.y_stride, j, n, more, ny[i]);
        load_group<MODE>(static_cast<const G*>(p.dh) + r * d, j, p.dh != nullptr ? n : 0, more && p.dh != nullptr, ng[i]);
        load_group<MODE>(static_cast<const X*>(p.ds) + r * d, j, p.ds != nullptr ? n : 0, more && p.ds != nullptr, nds[i]);
      }
    };
    fetch(row);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = group_at<TPR, 8>(i, off);
      w[i] = columns<MODE>(p.weight, p.weight_bf16, j, d);
      a[i] = mul(columns<MODE>(p.post_weight, p.post_bf16, j, d), factor);
      if (p.gate != nullptr && !own_gate) a[i] = mul(a[i], columns<MODE>(gate_row(p.gate, p.gate_bf16, gate, d), p.gate_bf16, j, d));
      u[i] = all8(0.f);
    }
    for (; row - group % PER_WARP < end; row += step) {
      const int n = row < end ? d : 0;
      const bool more = (p.rows - 1 - row) * d >= 7;
      const float r1 = nr.x, r2 = nr.y;
      V8 yh[NV], sh[NV], g[NV], dt[NV];
      uint4 words[NV];
      float2 acc = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = group_at<TPR, 8>(i, off);
        yh[i] = mul(values<MODE>(ny[i], j, n), r1);
        V8 b = mul(yh[i], a[i]);
        if (own_gate) b = mul(b, gate_values<MODE>(p.gate, p.gate_bf16, row, j, n, d, more));
        if (drops) {
          words[i] = drop_words(p.drop, seed, static_cast<uint64_t>(row * d + j) >> 3);
          b = kept(b, words[i], least);
        }
        sh[i] = mul(fma(values<MODE>(nx[i], j, n), p.alpha, b), r2);
        g[i] = values<MODE>(ng[i], j, n);
        dw[i] = fma(g[i], sh[i], dw[i]);
        g[i] = mul(g[i], w[i]);
        dot(acc, g[i], sh[i]);
        dt[i] = values<MODE>(nds[i], j, n);
      }
      if (row + step - group % PER_WARP < end) fetch(row + step);
      float sum[1] = {acc.x + acc.y};
      row_reduce<TPR, false>(sum, red[0]);
      const float c1 = -sum[0] * over;
      acc = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = group_at<TPR, 8>(i, off);
        dt[i] = fma(fma(sh[i], c1, g[i]), r2, dt[i]);
        if (p.dx != nullptr) put<MODE>(static_cast<X*>(p.dx) + row * d, j, n, mul(dt[i], p.alpha));
        if (drops) dt[i] = kept(dt[i], words[i], least);
        g[i] = mul(dt[i], a[i]);
        if (own_gate) {
          // The gate's own gradient (a is post_weight here), and the gate goes into the other two.
          const V8 gv = gate_values<MODE>(p.gate, p.gate_bf16, row, j, n, d, more);
          const V8 dg = mul(g[i], yh[i]);
          if (p.d_gate != nullptr) {
            if (p.gate_bf16)
              put<MODE>(static_cast<bf16*>(p.d_gate) + row * d, j, n, dg);
            else
              put<MODE>(static_cast<float*>(p.d_gate) + row * d, j, n, dg);
          }
          g[i] = mul(g[i], gv);
          dt[i] = mul(dt[i], gv);
        }
        u[i] = fma(dt[i], yh[i], u[i]);
        dot(acc, g[i], yh[i]);
      }
      sum[0] = acc.x + acc.y;
      row_reduce<TPR, false>(sum, red[1]);
      const float c2 = -sum[0] * over;
      if (p.dy != nullptr) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          put<MODE>(static_cast<Y*>(p.dy) + row * d, group_at<TPR, 8>(i, off), n, mul(fma(yh[i], c2, g[i]), r1));
      }
    }
    if (p.part_u != nullptr) leave(u, factor, p.part_u + static_cast<int64_t>(item) * d);
  }
  if (p.part_w != nullptr) leave(dw, 1.f, p.part_w + static_cast<int64_t>(blockIdx.x) * d);
}

template <class X, class Y, class G, int MODE>
cudaError_t go_branch_bwd(const BranchBwdParams& p, cudaStream_t st) {
  return branch_bwd_width(room_of(MODE, p.d), [&](auto tpr, auto nv) {
    constexpr int TPR = decltype(tpr)::value;
    const size_t smem = block_of(TPR) > TPR ? block_of(TPR) / TPR * sizeof(float) * static_cast<size_t>(p.d) : 0;
    branch_bwd_kernel<X, Y, G, TPR, decltype(nv)::value, MODE><<<p.blocks, block_of(TPR), smem, st>>>(p);
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
