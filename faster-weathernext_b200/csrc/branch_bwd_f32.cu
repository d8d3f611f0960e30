// Gradient of the residual branch, float32 stream (branch_bwd.cuh); its launch shape, and the sums of the partials.
#include "branch_bwd.cuh"

namespace fwn {

namespace {

__device__ __forceinline__ float value_at(const void* p, bool is_bf16, int64_t i) {
  return is_bf16 ? __bfloat162float(static_cast<const bf16*>(p)[i]) : static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void put_at(void* p, bool is_bf16, int64_t i, float v) {
  if (is_bf16)
    static_cast<bf16*>(p)[i] = __float2bfloat16_rn(v);
  else
    static_cast<float*>(p)[i] = v;
}

// A block of W warps takes 8 columns, a warp four rows of partials at a time. blockIdx.y 0: the slices' partials of u, gate by
// gate (as many gates at once as leave each a power of two of the warps), to d_gate and, over the gates, to d_post_weight; 1:
// the blocks' partials of d_weight.
template <int W>
__global__ void __launch_bounds__(32 * W) branch_bwd_finish_kernel(const BranchBwdParams p) {
  __shared__ float red[W][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = blockIdx.x * 8 + (lane & 7), d = p.d;
  const bool in = j < d;
  const bool for_u = blockIdx.y == 0 && p.part_u != nullptr;
  const float* part = for_u ? p.part_u : p.part_w;
  const int gates = for_u ? p.gates : 1, rows = for_u ? p.slices : p.blocks;
  int per = W;  // warps of a gate
  while (per > 1 && W / per < gates) per >>= 1;
  const int at_once = W / per, sub = warp % per;
  const bool gated = for_u && p.gate != nullptr && !p.gate_values;
  const float pw = for_u && p.post_weight != nullptr && in ? value_at(p.post_weight, p.post_bf16, j) : 1.f;
  float total = 0.f;
  for (int g0 = 0; g0 < gates; g0 += at_once) {
    const int g = g0 + warp / per;
    float t = 0.f;
    if (in && g < gates) {
#pragma unroll 8
      for (int r = 4 * sub + (lane >> 3); r < rows; r += 4 * per) t += part[(static_cast<int64_t>(g) * rows + r) * d + j];
    }
    t += __shfl_xor_sync(0xffffffffu, t, 8);
    t += __shfl_xor_sync(0xffffffffu, t, 16);
    if (per > 1) {
      if (lane < 8) red[warp][lane] = t;
      __syncthreads();
      if (sub == 0 && lane < 8)
        for (int q = 1; q < per; ++q) t += red[warp + q][lane];
      __syncthreads();
    }
    if (sub == 0 && lane < 8 && in && g < gates) {
      const int64_t at = static_cast<int64_t>(g) * d + j;
      if (gated && p.d_gate != nullptr) put_at(p.d_gate, p.gate_bf16, at, t * pw);
      total += gated ? t * value_at(p.gate, p.gate_bf16, at) : t;
    }
  }
  if (lane < 8) red[warp][lane] = total;  // 0 where sub > 0
  __syncthreads();
  if (warp == 0 && lane < 8 && in) {
    for (int q = 1; q < W; ++q) total += red[q][lane];
    if (for_u) {
      if (p.d_post != nullptr) put_at(p.d_post, p.post_bf16, j, total);
    } else {
      put_at(p.d_weight, p.weight_bf16, j, total);
    }
  }
}

}  // namespace

void branch_bwd_shape(int64_t rows, int d, int gates, int sms, bool wide, int* slices, int* blocks) {
  const int mode = wide ? kWide : kShift;
  const int room = branch_room(mode, d);
  branch_bwd_width(room, [&](auto tpr, auto maxt) {
    constexpr int TPR = decltype(tpr)::value, MAXT = decltype(maxt)::value, GROUPS = groups_of<TPR>();
    const int resident = sms * (branch_bwd_resident(MAXT) / branch_bwd_threads(TPR, MAXT, room));
    const int64_t most = (rows / gates + GROUPS - 1) / GROUPS;  // slices of a gate with a row each
    int64_t s = std::max<int64_t>(1, std::min<int64_t>(most, (resident + gates - 1) / gates));
    // kShift: the rows of a group start off alike, eight (or a multiple) apart, unless it has one row.
    if (!wide && GROUPS < 8) s = std::min<int64_t>(most, (s + 7) / 8 * 8);
    *slices = static_cast<int>(s);
    const int64_t items = s * gates;
    *blocks = static_cast<int>(wide ? std::min<int64_t>(items, resident) : items);
    return cudaSuccess;
  });
}

cudaError_t launch_branch_bwd_f32(const BranchBwdParams& p, cudaStream_t st) {
  return p.y_bf16 ? branch_bwd_by<float, bf16>(p, st) : branch_bwd_by<float, float>(p, st);
}

cudaError_t launch_branch_bwd_finish(const BranchBwdParams& p, cudaStream_t st) {
  const int sums = (p.part_u != nullptr ? 1 : 0) + (p.part_w != nullptr ? 1 : 0);
  if (sums == 0) return cudaSuccess;
  const dim3 grid(static_cast<unsigned>((p.d + 7) / 8), static_cast<unsigned>(sums));
  // Narrow rows have few blocks of many partials each, wide ones many of few.
  if (p.d <= 1024)
    branch_bwd_finish_kernel<32><<<grid, 1024, 0, st>>>(p);
  else
    branch_bwd_finish_kernel<8><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace fwn
