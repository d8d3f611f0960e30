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
// in order by branch_bwd_finish: no atomics, the same bits every time. Measured at 163,848 x 512, float32 stream, bf16 branch
// (of the measured copy rate): 230 us (1.00), with dropout 245 (0.94; bf16 stream 206, 0.75), and 7 for the sums; 40,962 x
// 2,048 233 (0.99); 163,848 x 333 247 (0.61).
//
// The gradient of s alone (no dh, G = none_t) does not depend on s: dt = ds, and x and rstd(s), which may hold anything then,
// take no part. A kernel of its own: a condition in the loop cost the other up to 29 % (163,848 x 512 230 -> 240 us, bf16
// stream with dropout 206 -> 245, 20,481 x 4,096 264 -> 339).
#pragma once

#include "branch_rows.cuh"

namespace fwn {

namespace {

// Threads of a row, eight values each: up to 256 values a warp or less, above them a block of as many warps as the row needs
// (of MAXT threads at most). Sixteen values a thread took as long at 512 (236 us) and longer with dropout (262 against 244):
// eight warps a SM left the exchanges between.
template <class F>
cudaError_t branch_bwd_width(int room, F f) {
  using std::integral_constant;
#define FWN_ROW(TPR, MAXT) \
  if (room <= (TPR > 0 ? TPR : MAXT) * 8) return f(integral_constant<int, TPR>(), integral_constant<int, MAXT>())
  FWN_ROW(8, 256);
  FWN_ROW(16, 256);
  FWN_ROW(32, 256);
  FWN_ROW(0, 128);
  FWN_ROW(0, 256);
  FWN_ROW(0, 512);
  FWN_ROW(0, 1024);
#undef FWN_ROW
  return cudaErrorInvalidValue;
}
constexpr int branch_bwd_resident(int maxt) { return maxt > 512 ? maxt : 512; }  // threads of an SM
__host__ __device__ constexpr int branch_bwd_threads(int tpr, int maxt, int room) { return tpr > 0 ? maxt : (room + 255) / 256 * 32; }

// G: dh's type, none_t without one.
template <class X, class Y, class G, int TPR, int MAXT, int MODE>
__global__ void __launch_bounds__(MAXT, branch_bwd_resident(MAXT) / MAXT) branch_bwd_kernel(const BranchBwdParams p) {
  constexpr int GROUPS = groups_of<TPR>(), PER_WARP = per_warp<TPR>();
  constexpr bool NORMED = !is_none<G>;
  extern __shared__ float part_smem[];  // more than one group: a row of d each
  __shared__ __align__(16) float red[2][32];
  clear_red<TPR>(red);
  const int d = p.d, group = TPR > 0 ? threadIdx.x / (TPR > 0 ? TPR : 1) : 0;
  const float over = 1.f / static_cast<float>(d);
  const bool drops = p.drop.threshold > 0, own_gate = p.gate_values;
  const uint32_t least = drop_least(p.drop);
  const float factor = drops ? p.drop.factor : 1.f;
  const uint64_t seed = drops ? drop_seed(p.drop) : 0;
  const int64_t span = p.gates > 1 ? p.gate_span : p.rows, step = static_cast<int64_t>(p.slices) * GROUPS;
  const int64_t whole = whole_rows(p.rows, d);
  V8 dw = all8(0.f);
  int j = column_of<TPR>(0, 0);
  // A block's row of partials: its groups' sums, added in order.
  auto leave = [&](const V8& v, float scale, float* to) {
    float* mine = GROUPS > 1 ? part_smem + group * d : to;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (j + e >= 0 && j + e < d) mine[j + e] = at8(v, e) * scale;
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
    if (MODE == kShift) j = column_of<TPR>(0, static_cast<int>(row * d & 7));  // of all the item's rows; a block takes one item
    const Cut<MODE> cut(j, d);
    Raw<X, 8> nx, nds;
    Raw<Y, 8> ny;
    Raw<std::conditional_t<NORMED, G, bf16>, 8> ng;
    float2 nr;
    auto fetch = [&](int64_t r) {
      const int n = r < end ? d : 0;  // a row that is not there adds nothing
      nr = n > 0 ? __ldg(reinterpret_cast<const float2*>(p.rstd) + r) : make_float2(0.f, 0.f);
      const X *x = static_cast<const X*>(p.x) + r * p.x_stride, *ds = static_cast<const X*>(p.ds) + r * d;
      const Y* y = static_cast<const Y*>(p.y) + r * p.y_stride;
      if constexpr (MODE == kWide) {
        if constexpr (NORMED) grab<MODE>(x, j, n, true, nx);
        grab<MODE>(y, j, n, true, ny);
        if constexpr (NORMED) grab<MODE>(static_cast<const G*>(p.dh) + r * d, j, n, true, ng);
        grab<MODE>(ds, j, p.ds != nullptr ? n : 0, true, nds);
      } else {
        const bool there = n > 0, all = r < whole;
        if constexpr (NORMED) grab_shifted(x, j, d, there, all, nx);
        grab_shifted(y, j, d, there, all, ny);
        if constexpr (NORMED) grab_shifted(static_cast<const G*>(p.dh) + r * d, j, d, there, all, ng);
        grab_shifted(ds, j, d, there && p.ds != nullptr, all, nds);
      }
    };
    fetch(row);
    const V8 w = columns<MODE>(p.weight, p.weight_bf16, j, d);
    V8 a = mul(columns<MODE>(p.post_weight, p.post_bf16, j, d), factor);  // post_weight gate factor
    if (p.gate != nullptr && !own_gate) a = mul(a, columns<MODE>(gate_row(p.gate, p.gate_bf16, gate, d), p.gate_bf16, j, d));
    V8 u = all8(0.f);  // sums of db yhat, without the factor
    for (; row - group % PER_WARP < end; row += step) {
      const int n = row < end ? d : 0;
      const float r1 = nr.x, r2 = nr.y;
      const V8 yh = mul(values(ny, cut), r1);
      V8 b = mul(yh, a);
      if (own_gate) b = mul(b, gate_values<MODE>(p.gate, p.gate_bf16, row, j, d, n > 0, row < whole, cut));
      uint4 words;
      if (drops) {
        words = drop_words(p.drop, seed, static_cast<uint64_t>(row * d + j) >> 3);
        b = kept(b, words, least);
      }
      V8 g, sh, dt = values(nds, cut);
      if constexpr (NORMED) {
        sh = mul(fma(values(nx, cut), p.alpha, b), r2);
        g = values(ng, cut);
      }
      if (row + step - group % PER_WARP < end) fetch(row + step);
      float2 acc = make_float2(0.f, 0.f);
      if constexpr (NORMED) {
        dw = fma(g, sh, dw);
        g = mul(g, w);
        dot(acc, g, sh);
        const float c1 = -over_row<TPR, false>(acc.x + acc.y, red[0]) * over;
        dt = fma(fma(sh, c1, g), r2, dt);
      } else if constexpr (TPR == 0) {
        __syncthreads();  // red[1] was read, which the other reduction's barrier orders otherwise
      }
      if (p.dx != nullptr) put<MODE>(static_cast<X*>(p.dx) + row * d, j, n, mul(dt, p.alpha));
      if (drops) dt = kept(dt, words, least);
      g = mul(dt, a);
      if (own_gate) {
        // The gate's own gradient (a is post_weight here), and the gate goes into the other two.
        const V8 gv = gate_values<MODE>(p.gate, p.gate_bf16, row, j, d, n > 0, row < whole, cut), dg = mul(g, yh);
        if (p.d_gate != nullptr) {
          if (p.gate_bf16)
            put<MODE>(static_cast<bf16*>(p.d_gate) + row * d, j, n, dg);
          else
            put<MODE>(static_cast<float*>(p.d_gate) + row * d, j, n, dg);
        }
        g = mul(g, gv);
        dt = mul(dt, gv);
      }
      u = fma(dt, yh, u);
      acc = make_float2(0.f, 0.f);
      dot(acc, g, yh);
      const float c2 = -over_row<TPR, false>(acc.x + acc.y, red[1]) * over;
      if (p.dy != nullptr) put<MODE>(static_cast<Y*>(p.dy) + row * d, j, n, mul(fma(yh, c2, g), r1));
    }
    if (p.part_u != nullptr) leave(u, factor, p.part_u + static_cast<int64_t>(item) * d);
  }
  if (p.part_w != nullptr) leave(dw, 1.f, p.part_w + static_cast<int64_t>(blockIdx.x) * d);
}

template <class X, class Y, class G, int MODE>
cudaError_t go_branch_bwd(const BranchBwdParams& p, cudaStream_t st) {
  const int room = branch_room(MODE, p.d);
  return branch_bwd_width(room, [&](auto tpr, auto maxt) {
    constexpr int TPR = decltype(tpr)::value, MAXT = decltype(maxt)::value, GROUPS = groups_of<TPR>();
    const size_t smem = GROUPS > 1 ? GROUPS * sizeof(float) * static_cast<size_t>(p.d) : 0;
    branch_bwd_kernel<X, Y, G, TPR, MAXT, MODE><<<p.blocks, branch_bwd_threads(TPR, MAXT, room), smem, st>>>(p);
    return cudaGetLastError();
  });
}
template <class X, class Y>
cudaError_t branch_bwd_by(const BranchBwdParams& p, cudaStream_t st) {
  if (p.dh == nullptr) return p.wide ? go_branch_bwd<X, Y, none_t, kWide>(p, st) : go_branch_bwd<X, Y, none_t, kShift>(p, st);
  if (p.dh_bf16) return p.wide ? go_branch_bwd<X, Y, bf16, kWide>(p, st) : go_branch_bwd<X, Y, bf16, kShift>(p, st);
  return p.wide ? go_branch_bwd<X, Y, float, kWide>(p, st) : go_branch_bwd<X, Y, float, kShift>(p, st);
}

}  // namespace

}  // namespace fwn
