// Products grouped by expert: what surrounds the tensor-core kernel (linear_tile.cuh): the experts' tensor maps, few rows,
// casts and sums.
//
// Rows offsets[e] to offsets[e + 1] of a tensor are expert e's. The offsets are on the device, where a router left them, and
// no call waits for them: group_setup_kernel counts the tiles before each expert, and gives every expert tensor maps of its
// own, the call's maps with their rows ending at the expert's last. The tensor core's kernel then needs no masks: loads past
// an expert's rows bring zeros (which a sum over rows adds), stores past them are dropped, and the rows behind, which may
// hold anything, are neither read nor written. Padding every expert to whole tiles instead costs a copy of the operand.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#define g_device_error g_grouped_device_error
#include "grouped.cuh"
#include "linear_tile.cuh"

namespace fwn {

namespace {

__device__ __forceinline__ int clamped(int v, int64_t m) { return static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(v), m))); }

// The row after expert g - 1's last (offsets[g] in order): the largest of the given ones up to g, by a warp.
__device__ __forceinline__ int end_before(const int32_t* given, int g, int64_t m) {
  int v = 0;
  for (int i = threadIdx.x & 31; i <= g; i += 32) v = max(v, clamped(__ldg(given + i), m));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Zeros to [begin, end) bytes of p by the threads of `blocks` blocks; all even numbers.
__device__ void clear_bytes(uint8_t* p, int64_t begin, int64_t end, int block, int blocks) {
  const int64_t id = static_cast<int64_t>(block) * blockDim.x + threadIdx.x, threads = static_cast<int64_t>(blocks) * blockDim.x;
  const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(p) & 15);
  const int64_t first = min(end, (begin + off + 15) / 16 * 16 - off), last = max(first, (end + off) / 16 * 16 - off);
  for (int64_t i = first + id * 16; i < last; i += threads * 16) *reinterpret_cast<uint4*>(p + i) = make_uint4(0, 0, 0, 0);
  for (int64_t i = begin + id * 2; i < first; i += threads * 2) *reinterpret_cast<uint16_t*>(p + i) = 0;
  for (int64_t i = last + id * 2; i < end; i += threads * 2) *reinterpret_cast<uint16_t*>(p + i) = 0;
}

constexpr int kClearBlocks = 64;

// Block 0: offsets and counts; the next `map_blocks`: a warp for each map of each expert; the others: rows of no expert.
__global__ void __launch_bounds__(1024) group_setup_kernel(const GroupSetup s, const __grid_constant__ GroupMaps maps, int map_blocks) {
  const int t = threadIdx.x, warp = t >> 5;
  if (blockIdx.x == 0) {
    __shared__ int warps[2][32], ends[1024];
    const int lane = t & 31;
    // Largest offset so far, then numbers of tiles before: scans over the 1,024 threads (`flip`: two scans' own warps[]).
    auto scan = [&](int v, bool most, int flip) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = most ? max(v, u) : v + u;
      }
      if (lane == 31) warps[flip][warp] = v;
      __syncthreads();
      int before = lane < warp ? warps[flip][lane] : 0;  // offsets and numbers are not negative
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const int u = __shfl_xor_sync(0xffffffffu, before, o);
        before = most ? max(before, u) : before + u;
      }
      return most ? max(v, before) : v + before;
    };
    const int given = t <= s.groups ? __ldg(s.given + t) : 0;
    const int mine = scan(clamped(given, s.m), true, 0);
    if (t <= s.groups) {
      s.offsets[t] = mine;
      if (mine != given) atomicOr(&g_device_error, 0x400u);  // out of order or of the tensor
    }
    ends[t] = mine;
    __syncthreads();
    const int rows = t < s.groups ? ends[t + 1] - mine : 0;
#pragma unroll
    for (int q = 0; q < kGroupFirsts; ++q) {
      if (s.first[q] == nullptr) continue;
      const int tiles = t < s.groups ? group_tiles(rows, s.unit[q]) : 0;
      const int upto = scan(tiles, false, (q + 1) & 1);
      if (t < s.groups) s.first[q][t] = upto - tiles;
      if (t == s.groups) s.first[q][t] = upto;  // tiles is 0 here
    }
  } else if (static_cast<int>(blockIdx.x) <= map_blocks) {
    __shared__ __align__(128) uint8_t copy[32][128];
    const int i = (blockIdx.x - 1) * 32 + warp;
    if (i >= s.n_maps * s.groups) return;  // whole warps
    const int q = i / s.groups, g = i % s.groups;
    const int end = end_before(s.given, g + 1, s.m);
    const uint32_t at = smem_u32(copy[warp]);
    reinterpret_cast<uint32_t*>(copy[warp])[t & 31] = reinterpret_cast<const uint32_t*>(&maps.map[q])[t & 31];
    __syncwarp();
    if ((t & 31) == 0)
      asm volatile("tensormap.replace.tile.global_dim.shared::cta.b1024.b32 [%0], 1, %1;" ::"r"(at), "r"(max(1, end)) : "memory");
    __syncwarp();
    asm volatile("tensormap.cp_fenceproxy.global.shared::cta.tensormap::generic.release.gpu.sync.aligned [%0], [%1], 128;"
                 ::"l"(reinterpret_cast<uint64_t>(s.maps + i)), "r"(at)
                 : "memory");
  } else {  // launched where there is a tensor to clear
    const int first = end_before(s.given, 0, s.m), last = end_before(s.given, s.groups, s.m);
    const int block = blockIdx.x - 1 - map_blocks;
    uint8_t* p = static_cast<uint8_t*>(s.clear);
    clear_bytes(p, 0, first * s.clear_row, block, kClearBlocks);
    clear_bytes(p, last * s.clear_row, s.m * s.clear_row, block, kClearBlocks);
  }
}

// Few rows: a warp per output column and run of rows of one expert (blockIdx.y: the run), lanes along k, so that the
// experts' weights stream through wide loads on as many SMs as there are columns.
template <int M, bool WIDE>
__global__ void __launch_bounds__(128) grouped_rows_kernel(const bf16* __restrict__ a, int64_t lda, const bf16* __restrict__ b,
                                                           int64_t ldb, int64_t b_stride, const int32_t* __restrict__ given,
                                                           int groups, const LinearParams p) {
  constexpr int V = WIDE ? 8 : 1;
  const int lane = threadIdx.x & 31, col = blockIdx.x * 4 + (threadIdx.x >> 5);
  // The expert of each row: row r is expert g's where offsets[g + 1] is the first to exceed r (-1: a row of none).
  const int m = static_cast<int>(p.m);
  int of[M];
#pragma unroll
  for (int r = 0; r < M; ++r) of[r] = -1;
  unsigned found = 0;
  bool wrong = false;
  int last = 0;
  for (int i0 = 0; i0 <= groups; i0 += 32) {
    const bool in = i0 + lane <= groups;
    const int v = in ? __ldg(given + i0 + lane) : INT_MAX;
    const int before = __shfl_up_sync(0xffffffffu, v, 1);
    wrong |= in && (v < 0 || v > m || v < (lane > 0 ? before : last));
    last = __shfl_sync(0xffffffffu, v, 31);
#pragma unroll
    for (int r = 0; r < M; ++r) {
      const unsigned over = __ballot_sync(0xffffffffu, in && v > r);
      if (over != 0 && !(found >> r & 1)) {
        found |= 1u << r;
        of[r] = i0 + __ffs(over) - 2;
      }
    }
  }
  if (wrong && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 32) atomicOr(&g_device_error, 0x400u);
  // The block's run of rows of one expert.
  int run = -1, g = -1, r0 = 0, r1 = 0;
#pragma unroll
  for (int r = 0; r < M; ++r) {
    if (r < m) {
      if (r == 0 || of[r] != of[r > 0 ? r - 1 : 0]) ++run;
      if (run == static_cast<int>(blockIdx.y)) {
        if (r1 == 0) r0 = r;
        r1 = r + 1;
        g = of[r];
      }
    }
  }
  if (r1 == 0 || col >= p.n) return;  // whole warps
  float acc[M];
#pragma unroll
  for (int r = 0; r < M; ++r) acc[r] = 0.f;
  if (g >= 0) {
    const bf16* brow = b + g * b_stride + col * ldb;
#pragma unroll 8
    for (int at = lane * V; at < p.k; at += 32 * V) {
      auto load = [](const bf16* src, float (&v)[V]) {
        if constexpr (WIDE) {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(src));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
          }
        } else {
          v[0] = __bfloat162float(*src);
        }
      };
      float w[V];
      load(brow + at, w);
#pragma unroll
      for (int r = 0; r < M; ++r) {
        if (r < r1 - r0) {
          float x[V];
          load(a + (r0 + r) * lda + at, x);
#pragma unroll
          for (int e = 0; e < V; ++e) acc[r] = fmaf(x[e], w[e], acc[r]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < M; ++r)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
  }
#pragma unroll
  for (int r = 0; r < M; ++r) {
    if (lane != r || r >= r1 - r0) continue;
    float v = acc[r];
    if (g >= 0) {
      const int64_t at = static_cast<int64_t>(g) * p.n + col;
      if (p.bias != nullptr)
        v += p.bias_bf16 ? __bfloat162float(static_cast<const bf16*>(p.bias)[at]) : static_cast<const float*>(p.bias)[at];
      v = p.act == 1 ? activate<1>(v) : p.act == 2 ? activate<2>(v) : v;
    }
    if (p.out_f32)
      static_cast<float*>(p.out)[(r0 + r) * p.ldo + col] = v;
    else
      static_cast<bf16*>(p.out)[(r0 + r) * p.ldo + col] = __float2bfloat16_rn(v);
  }
}

template <int M>
cudaError_t rows_go(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t b_stride, bool wide, const int32_t* given,
                    int groups, const LinearParams& p, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((p.n + 3) / 4), static_cast<unsigned>(p.m));
  const bf16 *x = static_cast<const bf16*>(a), *w = static_cast<const bf16*>(b);
  if (wide)
    grouped_rows_kernel<M, true><<<grid, 128, 0, st>>>(x, lda, w, ldb, b_stride, given, groups, p);
  else
    grouped_rows_kernel<M, false><<<grid, 128, 0, st>>>(x, lda, w, ldb, b_stride, given, groups, p);
  return cudaGetLastError();
}

// A block takes 32 V columns of a tile of kCastRows rows of an expert.
template <bool X32, int V>
__global__ void __launch_bounds__(256) grouped_cast_kernel(const void* __restrict__ x, int64_t ldx, int n, bf16* __restrict__ cast,
                                                           int64_t ldc, float* __restrict__ part, const GroupParams gp) {
  __shared__ float red[8][32 * V + 1];
  const int tile = blockIdx.x;
  if (tile >= __ldg(gp.first + gp.groups)) return;
  int lo = 0, hi = gp.groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(gp.first + mid) <= tile) lo = mid; else hi = mid;
  }
  const int64_t row0 = __ldg(gp.offsets + lo) + static_cast<int64_t>(tile - __ldg(gp.first + lo)) * kCastRows;
  const int64_t end = min(row0 + kCastRows, static_cast<int64_t>(__ldg(gp.offsets + lo + 1)));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (blockIdx.y * 32 + lane) * V;
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = 0.f;
  if (col < n) {
#pragma unroll 4
    for (int64_t r = row0 + warp; r < end; r += 8) {
      float v[V];
      if constexpr (V == 8) {
        if constexpr (X32) {
          const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(x) + r * ldx + col);
          const float4 a = __ldg(q), b = __ldg(q + 1);
          v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
          v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const bf16*>(x) + r * ldx + col));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
          }
        }
      } else {
        v[0] = X32 ? static_cast<const float*>(x)[r * ldx + col] : __bfloat162float(static_cast<const bf16*>(x)[r * ldx + col]);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] += v[e];
      if (cast != nullptr) {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          if constexpr (V == 1) {
            cast[r * ldc + col] = __float2bfloat16_rn(v[0]);
          } else {
            *reinterpret_cast<__nv_bfloat162*>(cast + r * ldc + col + e) = __floats2bfloat162_rn(v[e], v[e + 1]);
          }
        }
      }
    }
  }
  if (part == nullptr) return;
#pragma unroll
  for (int e = 0; e < V; ++e) red[warp][lane * V + e] = s[e];
  __syncthreads();
  for (int j = threadIdx.x; j < 32 * V; j += 256) {
    const int c = blockIdx.y * 32 * V + j;
    if (c < n) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) t += red[w][j];
      part[static_cast<int64_t>(tile) * n + c] = t;
    }
  }
}

// A block takes 32 V columns of an expert, its warps every W-th row of partials; their sums are added in order. Many experts
// have few rows each: 8 warps a block (64 even experts of 81,924 rows x 2,048: 8 to 11 us, 33 with 32 warps; where one expert
// has nine tenths of the rows, its blocks take 106).
template <int W, int V>
__global__ void __launch_bounds__(32 * W) grouped_column_sum_kernel(const float* __restrict__ part, const int32_t* __restrict__ first,
                                                                    int per, int n, void* __restrict__ out, bool out_bf16) {
  __shared__ float red[W][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = blockIdx.y;
  const int j0 = blockIdx.x * 32 * V, j = j0 + lane * V;
  const int64_t r0 = static_cast<int64_t>(__ldg(first + g)) * per, r1 = static_cast<int64_t>(__ldg(first + g + 1)) * per;
  float t[V];
#pragma unroll
  for (int e = 0; e < V; ++e) t[e] = 0.f;
  if (j < n) {
#pragma unroll 8
    for (int64_t r = r0 + warp; r < r1; r += W) {
      if constexpr (V == 4) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(part + r * n + j));
        t[0] += f.x;
        t[1] += f.y;
        t[2] += f.z;
        t[3] += f.w;
      } else {
        t[0] += __ldg(part + r * n + j);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) red[warp][lane * V + e] = t[e];
  __syncthreads();
  const int c = threadIdx.x;
  if (c >= 32 * V || j0 + c >= n) return;
  float sum = red[0][c];
#pragma unroll
  for (int w = 1; w < W; ++w) sum += red[w][c];
  const int64_t at = static_cast<int64_t>(g) * n + j0 + c;
  if (out_bf16)
    static_cast<bf16*>(out)[at] = __float2bfloat16_rn(sum);
  else
    static_cast<float*>(out)[at] = sum;
}

// A block takes an expert's row, four columns a thread at a time; the runs (in L2, just written) are added in order.
__global__ void __launch_bounds__(128) grouped_run_sum_kernel(const float* __restrict__ part, const int32_t* __restrict__ first,
                                                              int64_t rows, int n, int64_t ldp, bf16* __restrict__ out) {
  const int g = blockIdx.y;
  const int c0 = __ldg(first + g), c1 = __ldg(first + g + 1);
  const int64_t row = blockIdx.x;
  for (int j = threadIdx.x * 4; j < n; j += 512) {
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = c0; c < c1; ++c) {
      const float4 v = *reinterpret_cast<const float4*>(part + (c * rows + row) * ldp + j);
      t.x += v.x;
      t.y += v.y;
      t.z += v.z;
      t.w += v.w;
    }
    bf16* to = out + (g * rows + row) * n + j;
    const float u[4] = {t.x, t.y, t.z, t.w};
    if (n % 4 == 0 && reinterpret_cast<uintptr_t>(to) % 8 == 0) {
      *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(u[0], u[1]), pack_bf16(u[2], u[3]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j + e < n) to[e] = __float2bfloat16_rn(u[e]);
    }
  }
}

}  // namespace

cudaError_t launch_group_setup(const GroupSetup& s, const GroupMaps& maps, cudaStream_t st) {
  const int map_blocks = (s.n_maps * s.groups + 31) / 32;
  group_setup_kernel<<<1 + map_blocks + (s.clear != nullptr ? kClearBlocks : 0), 1024, 0, st>>>(s, maps, map_blocks);
  return cudaGetLastError();
}

cudaError_t launch_grouped_rows(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t b_stride, bool wide,
                                const int32_t* given, int groups, const LinearParams& p, cudaStream_t st) {
  if (p.m <= 1) return rows_go<1>(a, lda, b, ldb, b_stride, wide, given, groups, p, st);
  if (p.m <= 2) return rows_go<2>(a, lda, b, ldb, b_stride, wide, given, groups, p, st);
  if (p.m <= 4) return rows_go<4>(a, lda, b, ldb, b_stride, wide, given, groups, p, st);
  return rows_go<kLinearRowsMax>(a, lda, b, ldb, b_stride, wide, given, groups, p, st);
}

cudaError_t launch_grouped_cast(const void* x, bool x_f32, int64_t ldx, int n, void* cast, int64_t ldc, float* part,
                                const GroupParams& g, int64_t most, bool wide, cudaStream_t st) {
  const int v = wide ? 8 : 1;
  const dim3 grid(static_cast<unsigned>(most), static_cast<unsigned>((n + 32 * v - 1) / (32 * v)));
  auto* c = static_cast<bf16*>(cast);
  if (x_f32) {
    if (wide) grouped_cast_kernel<true, 8><<<grid, 256, 0, st>>>(x, ldx, n, c, ldc, part, g);
    else grouped_cast_kernel<true, 1><<<grid, 256, 0, st>>>(x, ldx, n, c, ldc, part, g);
  } else {
    if (wide) grouped_cast_kernel<false, 8><<<grid, 256, 0, st>>>(x, ldx, n, c, ldc, part, g);
    else grouped_cast_kernel<false, 1><<<grid, 256, 0, st>>>(x, ldx, n, c, ldc, part, g);
  }
  return cudaGetLastError();
}

cudaError_t launch_grouped_column_sum(const float* part, const int32_t* first, int groups, int64_t most, int per, int n, void* out,
                                      bool out_bf16, cudaStream_t st) {
  auto go = [&](auto kernel, int warps, int cols) {
    const dim3 grid(static_cast<unsigned>((n + cols - 1) / cols), static_cast<unsigned>(groups));
    kernel<<<grid, 32 * warps, 0, st>>>(part, first, per, n, out, out_bf16);
    return cudaGetLastError();
  };
  // Four columns a lane (the partials start on 256 bytes) where a warp adds few rows, else four times the blocks: 2,048 columns
  // of 2 rows a warp 2.4 (one column a lane: 3.9) us, 5 rows 10.8 (14.3), 10 rows 11.2 (10.8), 20 rows 21.7 (8.9).
  const bool wide = n % 4 == 0 && most * per <= 8ll * groups * (groups >= 16 ? 8 : 32);
  if (groups >= 16) return wide ? go(grouped_column_sum_kernel<8, 4>, 8, 128) : go(grouped_column_sum_kernel<8, 1>, 8, 32);
  return wide ? go(grouped_column_sum_kernel<32, 4>, 32, 128) : go(grouped_column_sum_kernel<32, 1>, 32, 32);
}

cudaError_t launch_grouped_run_sum(const float* part, const int32_t* first, int groups, int64_t rows, int n, int64_t ldp,
                                   void* out, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(groups));
  grouped_run_sum_kernel<<<grid, 128, 0, st>>>(part, first, rows, n, ldp, static_cast<bf16*>(out));
  return cudaGetLastError();
}

cudaError_t take_grouped_error(unsigned int* word) {
  cudaError_t e = cudaMemcpyFromSymbol(word, g_device_error, sizeof(*word));
  if (e != cudaSuccess) return e;
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
}

}  // namespace fwn
