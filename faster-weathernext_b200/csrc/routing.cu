// Routing of rows to experts: the largest logits of each row and their softmax, the rows in the experts' order (a stable
// counting sort), and the ways there and back with their gradients.
//
// Bound: HBM for the rows' ways (a row is read once and written to its `top` places, or the other way round; going by the
// sorted rows instead would read a row `top` times): 81,924 x 512 bf16 to two of eight experts there 41 us (0.94 of the copy
// rate), back 43 (0.90), the gradient of the way back 68 (0.94). Launches for the sort: one for few rows, else three (choice
// and counts per block, prefixes over the blocks, places): 18 us. No atomics decide an order: the same bits every time.
#include <algorithm>

#include "rms_rows.cuh"
#include "routing.cuh"

namespace fwn {

__device__ unsigned int g_routing_device_error = 0;

namespace {

// A logit as a number that orders as the choice does (NaN largest, -0 as 0; 0 is below every logit's), and with its place:
// the lower expert of equal logits is the larger.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return v != v ? 0xFFFFFFFFu : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long rank_of(float v, int e) {
  return static_cast<unsigned long long>(key_of(v)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(e));
}
__device__ __forceinline__ int expert_of(unsigned long long r) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(r)); }
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);  // NaN's key gives a NaN
}

// The block's rows: LPR lanes a row, NV logits a lane; `hist` [experts] counts their choices.
template <class T, int LPR, int NV>
__device__ void choose(const RouteParams& p, int64_t first, int* hist) {
  const int lane = threadIdx.x & (LPR - 1), per = blockDim.x / LPR;
  const T* logits = static_cast<const T*>(p.logits);
  const int rows = static_cast<int>(min(static_cast<int64_t>(kRouteRows), p.rows - first));
  // Whole warps go on while the first of their rows is there.
  for (int r = threadIdx.x / LPR; r - static_cast<int>(threadIdx.x & 31) / LPR < rows; r += per) {
    const int64_t row = first + r;
    const bool in = row < p.rows;
    unsigned long long keys[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = i * LPR + lane;
      keys[i] = in && e < p.experts ? rank_of(static_cast<float>(logits[row * p.stride + e]), e) : 0ull;
    }
    float top = 0.f, sum = 0.f, mine[kRouteTopMax / LPR + 1];  // choice j is lane j % LPR's
    int who[kRouteTopMax / LPR + 1];
#pragma unroll
    for (int j0 = 0; j0 < kRouteTopMax / LPR + 1; ++j0) {
      mine[j0] = 0.f;
      who[j0] = 0;
    }
#pragma unroll 1
    for (int j = 0; j < p.top; ++j) {
      unsigned long long best = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) best = max(best, keys[i]);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
#pragma unroll
      for (int i = 0; i < NV; ++i) keys[i] = keys[i] == best ? 0ull : keys[i];
      const float v = logit_of(static_cast<uint32_t>(best >> 32));
      if (j == 0) top = v;
      // A row whose logits are all -infinity: weights 0.
      const float w = top == -INFINITY ? 0.f : expf(v - top);
      sum += w;
#pragma unroll
      for (int j0 = 0; j0 < kRouteTopMax / LPR + 1; ++j0) {
        if (j == j0 * LPR + lane) {
          mine[j0] = w;
          who[j0] = expert_of(best);
        }
      }
    }
#pragma unroll
    for (int j0 = 0; j0 < kRouteTopMax / LPR + 1; ++j0) {
      const int j = j0 * LPR + lane;
      if (in && j < p.top) {
        p.chosen[row * p.top + j] = who[j0];
        p.weights[row * p.top + j] = top == -INFINITY ? 0.f : mine[j0] / sum;
        atomicAdd(hist + who[j0], 1);
      }
    }
  }
}

// The places of the block's pairs (row, choice) in their order: `base` [experts] is where the block's first of each expert
// goes; `count` [8, experts] is the warps' workspace. A warp takes adjacent pairs.
__device__ void place(const RouteParams& p, int64_t first, const int* base, int* count) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pairs = static_cast<int>(min(static_cast<int64_t>(kRouteRows), p.rows - first)) * p.top;
  const int each = (pairs + 255) / 256 * 32;
  const int begin = warp * each, end = min(pairs, begin + each);
  int* mine = count + warp * p.experts;
  for (int i = threadIdx.x; i < 8 * p.experts; i += blockDim.x) count[i] = 0;
  __syncthreads();
  for (int pass = 0; pass < 2; ++pass) {
    for (int i = begin; i < end; i += 32) {
      const bool in = i + lane < end;
      const int64_t pair = first * p.top + i + lane;
      const int e = in ? p.chosen[pair] : -1;
      const unsigned same = __match_any_sync(0xffffffffu, e);
      const int rank = __popc(same & ((1u << lane) - 1u));
      const int at = in ? mine[e] : 0;
      __syncwarp();
      if (in && rank == 0) mine[e] = at + __popc(same);
      __syncwarp();
      if (pass == 1 && in) {
        p.position[pair] = at + rank;
        p.order[at + rank] = static_cast<int32_t>(pair);
      }
    }
    __syncthreads();
    if (pass == 0) {
      for (int e = threadIdx.x; e < p.experts; e += blockDim.x) {
        int at = base[e];
        for (int w = 0; w < 8; ++w) {
          const int n = count[w * p.experts + e];
          count[w * p.experts + e] = at;
          at += n;
        }
      }
      __syncthreads();
    }
  }
}

// Exclusive prefixes of total [n] (n <= 1,023) by a block of 256 threads, with the sum behind them: out [n + 1].
__device__ void prefixes(const int* total, int n, int* out) {
  __shared__ int sums[8];
  const int t = threadIdx.x, lane = t & 31;
  int v[4], s = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = 4 * t + i < n ? total[4 * t + i] : 0;
    s += v[i];
  }
  int upto = s;  // of the warp's threads so far
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (lane == 31) sums[t >> 5] = upto;
  __syncthreads();
  int at = upto - s;
  for (int w = 0; w < t >> 5; ++w) at += sums[w];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (4 * t + i <= n) out[4 * t + i] = at;
    at += v[i];
  }
  __syncthreads();
}

// Few rows, one block's: choice, prefixes and places in this launch; several lanes a row.
template <class T, int LPR, int NV>
__global__ void __launch_bounds__(256) route_few_kernel(const RouteParams p) {
  extern __shared__ int route_smem[];  // hist [experts], prefixes [experts + 1], counts [8, experts]
  int* hist = route_smem;
  for (int e = threadIdx.x; e < p.experts; e += 256) hist[e] = 0;
  __syncthreads();
  choose<T, LPR, NV>(p, 0, hist);
  __syncthreads();
  int* at = hist + p.experts;
  prefixes(hist, p.experts, at);
  for (int e = threadIdx.x; e <= p.experts; e += 256) p.offsets[e] = at[e];
  place(p, 0, at, at + p.experts + 1);
}

// Many rows: a thread per row keeps its K largest in order, without exchanges; the logits come through shared memory, C
// experts of the block's rows at a time (81,924 rows x 64 experts, two of them: 36 us with a warp per row, each choice a
// maximum over the lanes, 94 us for eight; 12 and 25 so).
template <class T, int K, int C>
__global__ void __launch_bounds__(kRouteRows) route_choose_kernel(const RouteParams p) {
  __shared__ uint32_t keys[kRouteRows][C + 1];
  extern __shared__ int route_smem[];  // hist [experts]
  int* hist = route_smem;
  const int t = threadIdx.x;
  for (int e = t; e < p.experts; e += kRouteRows) hist[e] = 0;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRouteRows;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kRouteRows), p.rows - first));
  const T* logits = static_cast<const T*>(p.logits) + first * p.stride;
  uint32_t best[K];
  int who[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    best[j] = 0;
    who[j] = 0;
  }
  // The next experts' logits are on their way while some are gone through.
  T next[C];
  auto fetch = [&](int e0) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int r = (i * kRouteRows + t) / C, c = (i * kRouteRows + t) % C;
      next[i] = T(0.f);
      if (r < rows && e0 + c < p.experts) next[i] = logits[r * p.stride + e0 + c];
    }
  };
  fetch(0);
  for (int e0 = 0; e0 < p.experts; e0 += C) {
    const int n = min(C, p.experts - e0);
    if (e0 > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < C; ++i) keys[(i * kRouteRows + t) / C][(i * kRouteRows + t) % C] = key_of(static_cast<float>(next[i]));
    __syncthreads();
    if (e0 + C < p.experts) fetch(e0 + C);
    if (t < rows) {
#pragma unroll 4
      for (int c = 0; c < n; ++c) {
        const uint32_t key = keys[t][c];
        if (key <= best[K - 1]) continue;  // equal ones stay behind those before them
#pragma unroll
        for (int j = K - 1; j >= 0; --j) {
          const bool up = j > 0 && key > best[j > 0 ? j - 1 : 0], here = key > best[j];
          who[j] = up ? who[j > 0 ? j - 1 : 0] : here ? e0 + c : who[j];
          best[j] = up ? best[j > 0 ? j - 1 : 0] : here ? key : best[j];
        }
      }
    }
  }
  if (t < rows) {
    const float top = logit_of(best[0]);
    float w[K], sum = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      w[j] = j < p.top && top != -INFINITY ? expf(logit_of(best[j]) - top) : 0.f;  // all -infinity: weights 0
      sum += w[j];
    }
    const int64_t at = (first + t) * p.top;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (j < p.top) {
        p.chosen[at + j] = who[j];
        p.weights[at + j] = top == -INFINITY ? 0.f : w[j] / sum;
        atomicAdd(hist + who[j], 1);
      }
    }
  }
  __syncthreads();
  for (int e = t; e < p.experts; e += kRouteRows) p.counts[static_cast<int64_t>(e) * gridDim.x + blockIdx.x] = hist[e];
}

// A warp per expert: its blocks' counts become prefixes, and its total.
__global__ void __launch_bounds__(256) route_scan_kernel(const RouteParams p, int64_t blocks) {
  const int e = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (e >= p.experts) return;
  int32_t* c = p.counts + e * blocks;
  int total = 0;
  for (int64_t b0 = 0; b0 < blocks; b0 += 128) {
    int v[4], s = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = b0 + 4 * lane + i < blocks ? c[b0 + 4 * lane + i] : 0;
      s += v[i];
    }
    int upto = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    int at = total + upto - s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (b0 + 4 * lane + i < blocks) c[b0 + 4 * lane + i] = at;
      at += v[i];
    }
    total += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) p.totals[e] = total;
}

__global__ void __launch_bounds__(256) route_place_kernel(const RouteParams p) {
  extern __shared__ int route_smem[];  // prefixes [experts + 1], counts [8, experts]
  int* at = route_smem;
  prefixes(p.totals, p.experts, at);
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= p.experts; e += 256) p.offsets[e] = at[e];
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += 256) at[e] += p.counts[static_cast<int64_t>(e) * gridDim.x + blockIdx.x];
  __syncthreads();
  place(p, static_cast<int64_t>(blockIdx.x) * kRouteRows, at, at + p.experts + 1);
}

template <class F>
cudaError_t by_top(int top, F f) {
  using std::integral_constant;
  if (top <= 1) return f(integral_constant<int, 1>());
  if (top <= 2) return f(integral_constant<int, 2>());
  if (top <= 4) return f(integral_constant<int, 4>());
  if (top <= 8) return f(integral_constant<int, 8>());
  return f(integral_constant<int, kRouteTopMax>());
}

template <class T, int LPR, int NV>
cudaError_t few_go(const RouteParams& p, cudaStream_t st) {
  route_few_kernel<T, LPR, NV><<<1, 256, (10 * p.experts + 1) * sizeof(int), st>>>(p);
  return cudaGetLastError();
}
template <class T>
cudaError_t route_few(const RouteParams& p, cudaStream_t st) {
  if (p.experts <= 8) return few_go<T, 8, 1>(p, st);
  if (p.experts <= 16) return few_go<T, 16, 1>(p, st);
  if (p.experts <= 32) return few_go<T, 32, 1>(p, st);
  if (p.experts <= 64) return few_go<T, 32, 2>(p, st);
  if (p.experts <= 256) return few_go<T, 32, 8>(p, st);
  return few_go<T, 32, 32>(p, st);
}
template <class T>
cudaError_t route_many(const RouteParams& p, cudaStream_t st) {
  const int64_t blocks = route_blocks(p.rows);
  const size_t e = static_cast<size_t>(p.experts) * sizeof(int);
  cudaError_t err = by_top(p.top, [&](auto k) {
    constexpr int K = decltype(k)::value;
    if (p.experts <= 8)
      route_choose_kernel<T, K, 8><<<static_cast<unsigned>(blocks), kRouteRows, e, st>>>(p);
    else if (p.experts <= 16)
      route_choose_kernel<T, K, 16><<<static_cast<unsigned>(blocks), kRouteRows, e, st>>>(p);
    else
      route_choose_kernel<T, K, 32><<<static_cast<unsigned>(blocks), kRouteRows, e, st>>>(p);
    return cudaGetLastError();
  });
  if (err != cudaSuccess) return err;
  route_scan_kernel<<<(p.experts + 7) / 8, 256, 0, st>>>(p, blocks);
  route_place_kernel<<<static_cast<unsigned>(blocks), 256, 9 * e + sizeof(int), st>>>(p);
  return cudaGetLastError();
}

// d logit[chosen j] = w_j (d w_j - sum over i of w_i d w_i), 0 elsewhere: a block clears its rows, then a thread per row
// writes the chosen.
template <class T>
__global__ void __launch_bounds__(kRouteRows) route_bwd_kernel(const float* __restrict__ weights, const int32_t* __restrict__ chosen,
                                                               const float* __restrict__ d_weights, int64_t rows, int experts, int top,
                                                               T* __restrict__ d_logits, bool wide) {
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRouteRows, row = first + threadIdx.x;
  const int64_t n = min(static_cast<int64_t>(kRouteRows), rows - first) * experts;
  T* out = d_logits + first * experts;
  const int64_t wide_n = wide ? n / (16 / sizeof(T)) : 0;
  for (int64_t i = threadIdx.x; i < wide_n; i += kRouteRows) reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
  for (int64_t i = wide_n * (16 / sizeof(T)) + threadIdx.x; i < n; i += kRouteRows) out[i] = T(0.f);
  __syncthreads();
  if (row >= rows) return;
  float sum = 0.f;
  for (int j = 0; j < top; ++j) sum = fmaf(__ldg(weights + row * top + j), __ldg(d_weights + row * top + j), sum);
  for (int j = 0; j < top; ++j) {
    const float w = __ldg(weights + row * top + j), v = w == 0.f ? 0.f : w * (__ldg(d_weights + row * top + j) - sum);
    const int e = __ldg(chosen + row * top + j);
    T* to = out + static_cast<int64_t>(threadIdx.x) * experts + e;
    if (e < 0 || e >= experts) continue;  // not this routing's
    if constexpr (sizeof(T) == 2)
      *to = __float2bfloat16_rn(v);
    else
      *to = v;
  }
}

// ---- the rows' ways -------------------------------------------------------------------------------------------------

// The place of a pair, or -1 (reported) where it would lie outside.
__device__ __forceinline__ int64_t place_of(const RowMoveParams& p, int64_t row, int j) {
  const int32_t at = __ldg(p.position + row * p.top + j);
  if (at >= 0 && at < p.rows * p.top) return at;
  atomicOr(&g_routing_device_error, 0x400u);
  return -1;
}

// V values of a row: 8 (16 or 32 bytes), 2 (4 or 8) or 1.
template <class T, int V>
__device__ __forceinline__ void take(const T* p, Raw<T, V>& r) {
  if constexpr (V != 2) {
    load_raw(p, r);
  } else if constexpr (sizeof(T) == 4) {
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
    r.u[0] = u.x;
    r.u[1] = u.y;
  } else {
    r.u[0] = __ldg(reinterpret_cast<const unsigned int*>(p));
  }
}
template <class T, int V>
__device__ __forceinline__ void give(T* p, const float (&v)[V]) {
  if constexpr (V != 2) {
    store_vals(p, v);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  } else {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v[0], v[1]);
  }
}
// Accesses of a thread on their way: some 64 bytes, eight at most.
constexpr int at_once(int bytes) { return bytes >= 64 ? 1 : 64 / bytes > 8 ? 8 : 64 / bytes; }

// L lanes a row. DOTS: the products x . y of the row's places too. V values an access.
template <class T, int V, int L, int K, bool DOTS>
__global__ void __launch_bounds__(256) spread_kernel(const RowMoveParams p) {
  constexpr int U = DOTS ? (K >= 8 ? 1 : at_once((K + 1) * V * static_cast<int>(sizeof(T)) / 2)) : at_once(V * static_cast<int>(sizeof(T)));
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / L) + threadIdx.x / L;
  if (row >= p.rows) return;  // whole rows: their lanes exchange among themselves alone
  const int lane = threadIdx.x & (L - 1);
  const unsigned mine = L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1u) << (threadIdx.x & 31 & ~(L - 1));
  int64_t at[K];
  float w[K], dot[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    at[j] = j < p.top ? place_of(p, row, j) : -1;
    w[j] = p.weights != nullptr && j < p.top ? __ldg(p.weights + row * p.top + j) : 1.f;
    dot[j] = 0.f;
  }
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  for (int c0 = lane * V; c0 < p.d; c0 += L * V * U) {
    Raw<T, V> r[U], q[DOTS ? K : 1][DOTS ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * L * V;
      if (c < p.d) take(x + c, r[u]);
    }
    if constexpr (DOTS) {
#pragma unroll
      for (int j = 0; j < K; ++j)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = c0 + u * L * V;
          if (at[j] >= 0 && c < p.d) take(static_cast<const T*>(p.y) + at[j] * p.d + c, q[j][u]);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * L * V;
      if (c >= p.d) break;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if (at[j] < 0) continue;
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = raw_at(r[u], e);
        if constexpr (DOTS) {
#pragma unroll
          for (int e = 0; e < V; ++e) dot[j] = fmaf(v[e], raw_at(q[j][u], e), dot[j]);
        }
        if (p.weights != nullptr) {
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] *= w[j];
        }
        if (p.to != nullptr) give(static_cast<T*>(p.to) + at[j] * p.d + c, v);
      }
    }
  }
  if constexpr (DOTS) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(mine, dot[j], o);
      if (lane == j % L && j < p.top) p.dots[row * p.top + j] = dot[j];
    }
  }
}

template <class T, int V, int L, int K>
__global__ void __launch_bounds__(256) gather_kernel(const RowMoveParams p) {
  constexpr int U = at_once(K * V * static_cast<int>(sizeof(T)));
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / L) + threadIdx.x / L;
  if (row >= p.rows) return;
  const int lane = threadIdx.x & (L - 1);
  int64_t at[K];
  float w[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    at[j] = j < p.top ? place_of(p, row, j) : -1;
    w[j] = p.weights != nullptr && j < p.top ? __ldg(p.weights + row * p.top + j) : 1.f;
  }
  for (int c0 = lane * V; c0 < p.d; c0 += L * V * U) {
    Raw<T, V> q[K][U];
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + u * L * V;
        if (at[j] >= 0 && c < p.d) take(static_cast<const T*>(p.y) + at[j] * p.d + c, q[j][u]);
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * L * V;
      if (c >= p.d) break;
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if (at[j] < 0) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = fmaf(w[j], raw_at(q[j][u], e), v[e]);
      }
      give(static_cast<T*>(p.to) + row * p.d + c, v);
    }
  }
}

// Values an access by what every row of each tensor allows, and lanes a row by its accesses.
template <class T, class F>
cudaError_t by_row(const RowMoveParams& p, F f) {
  using std::integral_constant;
  if (p.wide) {
    if (p.d <= 64) return f(integral_constant<int, 8>(), integral_constant<int, 8>());
    if (p.d <= 128) return f(integral_constant<int, 8>(), integral_constant<int, 16>());
    return f(integral_constant<int, 8>(), integral_constant<int, 32>());
  }
  if (p.pairs) return f(integral_constant<int, 2>(), integral_constant<int, 32>());
  return f(integral_constant<int, 1>(), integral_constant<int, 32>());
}
template <class T>
cudaError_t spread_go(const RowMoveParams& p, cudaStream_t st) {
  return by_row<T>(p, [&](auto v, auto l) {
    return by_top(p.top, [&](auto k) {
      constexpr int V = decltype(v)::value, L = decltype(l)::value, K = decltype(k)::value;
      const unsigned blocks = static_cast<unsigned>((p.rows + 256 / L - 1) / (256 / L));
      if (p.dots != nullptr)
        spread_kernel<T, V, L, K, true><<<blocks, 256, 0, st>>>(p);
      else
        spread_kernel<T, V, L, K, false><<<blocks, 256, 0, st>>>(p);
      return cudaGetLastError();
    });
  });
}
template <class T>
cudaError_t gather_go(const RowMoveParams& p, cudaStream_t st) {
  return by_row<T>(p, [&](auto v, auto l) {
    return by_top(p.top, [&](auto k) {
      constexpr int V = decltype(v)::value, L = decltype(l)::value, K = decltype(k)::value;
      gather_kernel<T, V, L, K><<<static_cast<unsigned>((p.rows + 256 / L - 1) / (256 / L)), 256, 0, st>>>(p);
      return cudaGetLastError();
    });
  });
}

}  // namespace

cudaError_t launch_route(const RouteParams& p, cudaStream_t st) {
  if (route_blocks(p.rows) == 1) return p.bf16_logits ? route_few<bf16>(p, st) : route_few<float>(p, st);
  return p.bf16_logits ? route_many<bf16>(p, st) : route_many<float>(p, st);
}

cudaError_t launch_route_bwd(const float* weights, const int32_t* chosen, const float* d_weights, int64_t rows, int experts,
                             int top, void* d_logits, bool bf16_logits, cudaStream_t st) {
  const unsigned blocks = static_cast<unsigned>(route_blocks(rows));
  const bool wide = reinterpret_cast<uintptr_t>(d_logits) % 16 == 0;  // a block's rows start at multiples of 128 values
  if (bf16_logits)
    route_bwd_kernel<<<blocks, kRouteRows, 0, st>>>(weights, chosen, d_weights, rows, experts, top, static_cast<bf16*>(d_logits), wide);
  else
    route_bwd_kernel<<<blocks, kRouteRows, 0, st>>>(weights, chosen, d_weights, rows, experts, top, static_cast<float*>(d_logits), wide);
  return cudaGetLastError();
}

cudaError_t launch_spread(const RowMoveParams& p, cudaStream_t st) {
  return p.bf16_rows ? spread_go<bf16>(p, st) : spread_go<float>(p, st);
}
cudaError_t launch_gather(const RowMoveParams& p, cudaStream_t st) {
  return p.bf16_rows ? gather_go<bf16>(p, st) : gather_go<float>(p, st);
}

cudaError_t take_routing_error(unsigned int* word) {
  cudaError_t e = cudaMemcpyFromSymbol(word, g_routing_device_error, sizeof(*word));
  if (e != cudaSuccess) return e;
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_routing_device_error, &zero, sizeof(zero));
}

}  // namespace fwn
