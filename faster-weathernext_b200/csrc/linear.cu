// Projections: out = act(a b^T + bias) + residual over any m, n, k, bf16 or 8-bit operands, and what their gradients
// need.
//
// linear_tile_kernel, the tensor-core kernel (tcgen05, TMA, TMEM), takes every product of more than kLinearRowsMax
// rows: the forward, d_a = d_pre b, d_b = d_pre^T a (an operand's k or its m / n may be the contiguous dimension: both
// orders of the shared-memory descriptors), and d_pre = dy act'(a b^T + bias) with its column sums, which recomputes
// the pre-activation instead of keeping it. linear_rows_kernel takes the few rows of a serving call.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

// This translation unit's device error word.
#define g_device_error g_linear_device_error
#include "common.cuh"
#include "linear.cuh"

namespace fwn {

namespace {

using bf16 = __nv_bfloat16;

// ---- PTX helpers of this file --------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of `addr` (this CTA's shared memory) in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// No cluster-scope release: it orders tensor-memory reads, which tcgen05.fence has ordered before it, and took 1,000
// cycles behind the thread's outstanding stores.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Tile load; CG = 2: the barrier may be the pair's other CTA's (its bytes count there).
template <int CG>
__device__ __forceinline__ void tile_load(uint32_t dst, const void* tmap, int c0, int c1, uint32_t bar) {
  if constexpr (CG == 2) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
  }
}
__device__ __forceinline__ void tile_store(const void* tmap, int c0, int c1, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
               ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(src)
               : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// A bounded wait of a whole warp by polling (mbarrier.test_wait), for the producers and the MMA warp: 20.3 us at 10,242 x
// 512 x 2,048 against 21.2 with mbarrier.try_wait, which may suspend the warp. The epilogue's warps wait with try_wait.
__device__ __forceinline__ bool poll_wait(uint32_t bar, uint32_t parity, volatile int* abort) {
  auto attempt = [&] {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
  };
  bool ok = attempt();
  if (!ok) {
    unsigned long long t0 = 0;
    for (uint32_t i = 1; !(ok = attempt()); ++i) {
      if ((i & 255u) == 0u) {
        if (*abort) break;
        const unsigned long long t = globaltimer();
        if (t0 == 0) t0 = t;
        if (t - t0 > kWaitLimitNs) {
          *abort = 1;
          atomicOr(&g_device_error, 5u);
          break;
        }
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}
template <int CG>
__device__ __forceinline__ void tmem_alloc_cg(uint32_t dst, uint32_t cols) {
  if constexpr (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(dst, cols);
  }
}
template <int CG>
__device__ __forceinline__ void tmem_dealloc_cg(uint32_t addr, uint32_t cols) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
  else
    tmem_dealloc(addr, cols);
}
// D[tmem] (+)= A B^T from shared memory; CG = 2: this CTA's and its pair's A rows and B rows.
template <int CG, bool FP8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
#define FWN_MMA(GROUP, KIND)                                                                            \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                                        \
               "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, p;\n\t}" ::"r"(d),    \
               "l"(a), "l"(b), "r"(idesc), "r"(accumulate)                                              \
               : "memory")
  if constexpr (CG == 2) {
    if constexpr (FP8) FWN_MMA("2", "f8f6f4"); else FWN_MMA("2", "f16");
  } else {
    if constexpr (FP8) FWN_MMA("1", "f8f6f4"); else FWN_MMA("1", "f16");
  }
#undef FWN_MMA
}
// Arrive on `bar` (CG = 2: on the barrier at that offset in both CTAs) when the MMAs issued so far are complete.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"(static_cast<uint16_t>(3))
                 : "memory");
  else
    mma_commit(bar);
}

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- activations ---------------------------------------------------------------------------------------------------

constexpr float kGeluC0 = 0.7978845608028654f, kGeluC1 = 0.044715f, kLog2e = 1.4426950408889634f;

// GELU in its tanh form is x sigma(2 u), u = c0 (x + c1 x^3), swish x sigma(x): written through the logistic function
// sigma(z) = 1 / (1 + 2^-z') both keep their relative precision where they are small, which 1 + tanh does not.
// Coefficients of z' = -z log2(e) = x (p0 + p1 x^2).
template <int ACT>
struct Logistic {
  static constexpr float p0 = ACT == 1 ? -2.f * kLog2e * kGeluC0 : -kLog2e;
  static constexpr float p1 = ACT == 1 ? p0 * kGeluC1 : 0.f;
  // dz/dx = q0 + q1 x^2
  static constexpr float q0 = ACT == 1 ? 2.f * kGeluC0 : 1.f, q1 = ACT == 1 ? 3.f * kGeluC1 * q0 : 0.f;
  // Below `low`, where 2^z' is about 2^30, bf16 results are taken as those at `low` (-5.9e-9, for swish -1.6e-8), and so is
  // the slope (-4.7e-8, for swish -1.5e-8); above `high` the slope is 1 to float32's last bit.
  static constexpr float low = ACT == 1 ? -5.5f : -21.f, high = ACT == 1 ? 10.f : 40.f;
};
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// One value, to float32 precision over the whole range. -infinity counts as the lowest finite value, whose result is -0, the
// functions' limit, and what the clamp at `low` comes to in bf16 (x sigma would be infinity times 0).
template <int ACT>
__device__ __forceinline__ float activate(float x) {
  if constexpr (ACT == 0) return x;
  using L = Logistic<ACT>;
  x = max_nan(x, -3.402823466e38f);
  const float z = ACT == 1 ? x * fmaf(L::p1 * x, x, L::p0) : x * L::p0;
  return x * rcp(1.f + ex2(z));
}
__device__ __forceinline__ float2 pair(float a) { return make_float2(a, a); }
// Four values for a bf16 result. The special-function unit, not the FP32 pipe, bounds an epilogue of two calls a value
// (4,096 cycles for a 128 x 256 tile, as long as its MMAs at k = 512): the four denominators 1 + 2^z' (each at most 2^31,
// so that their product stays in float32) share one reciprocal, 1.25 calls a value, and the rest runs in pairs. A NaN must
// not reach that product, or three other columns would be NaN with it: the denominators take a minimum that drops it, and
// x (in the slope 2^z' too) carries it into its own result.
template <int ACT, bool SLOPE>
__device__ __forceinline__ void activate4(float* v) {
  using L = Logistic<ACT>;
  constexpr float kDenomMax = 2147483648.f;
  float2 x[2], d[2], e[2], xx[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[i] = make_float2(max_nan(v[2 * i], L::low), max_nan(v[2 * i + 1], L::low));
    if constexpr (SLOPE) x[i] = make_float2(min_nan(x[i].x, L::high), min_nan(x[i].y, L::high));
    float2 z;
    if constexpr (ACT == 1) {
      xx[i] = fmul2(x[i], x[i]);
      z = fmul2(x[i], ffma2(xx[i], pair(L::p1), pair(L::p0)));
    } else {
      z = fmul2(x[i], pair(L::p0));
    }
    e[i] = make_float2(ex2(z.x), ex2(z.y));
    d[i] = fadd2(make_float2(fminf(e[i].x, kDenomMax), fminf(e[i].y, kDenomMax)), pair(1.f));
  }
  const float2 m = fmul2(d[0], d[1]);
  const float r = rcp(m.x * m.y);
  const float2 n = fmul2(pair(r), make_float2(m.y, m.x));  // 1 / (d0 d2), 1 / (d1 d3)
  const float2 s[2] = {fmul2(n, d[1]), fmul2(n, d[0])};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float2 y;
    if constexpr (SLOPE) {
      // sigma + x sigma (1 - sigma) z_x = sigma (1 + (1 - sigma) x z_x), 1 - sigma = 2^z' sigma
      const float2 w = ACT == 1 ? fmul2(x[i], ffma2(xx[i], pair(L::q1), pair(L::q0))) : x[i];
      y = fmul2(s[i], ffma2(fmul2(e[i], s[i]), w, pair(1.f)));
    } else {
      y = fmul2(x[i], s[i]);
    }
    v[2 * i] = y.x;
    v[2 * i + 1] = y.y;
  }
}

// ---- tensor-core kernel --------------------------------------------------------------------------------------------

// Persistent; a CTA (CG = 1) or a pair of CTAs on two SMs (CG = 2) takes output tiles of 128 CG x BN, walked with n
// fastest so that the tiles in flight share their rows of a in L2. Warps:
//   0      TMA producer of a: 128 bytes of k (64 bf16, 128 e4m3) of 128 rows (b: BN / CG rows) per stage, or, with m
//          (n) contiguous, 64 rows of k by 64 columns, one box per 64;
//   1      MMA issuer (CG = 2: of the pair's first CTA, for both), into one of two TMEM accumulators;
//   2      the same producer for b (one lane issues a load in about 200 cycles; two loads a stage held the MMAs);
//   3      idle (it completes the warpgroup whose registers the epilogue takes);
//   4-     epilogue, 16 warps (8 on the small tiles): warp w reads TMEM lanes 32 (w % 4) + [0, 32) (rows) and 64 of
//          the tile's columns, in chunks of 128 bytes of a row; the residual (or dy) chunk arrives by TMA in the warp's
//          slot, the result replaces it there and leaves by TMA, and a tile's epilogue overlaps the next tile's MMAs.
//          With 8 warps the chain TMEM -> arithmetic -> shared memory -> store of two warps per scheduler left it idle.
// Ragged edges: TMA fills rows and columns past the tensors with zeros and clips stores. Why a pair on 256 x 256: per
// 64 of k an SM then takes in 32 KB for 512 cycles of MMA, half the L2 traffic per FLOP of 128 x 128 and two thirds of
// 128 x 256. The small tiles spread products of few rows over the SMs. Why chunks of 128-byte rows: a TMA store of 32
// rows took about 200 cycles whether its rows had 64 bytes or 128, which held a 163,848 x 2,048 bf16 result to 226 us.
//
// float32 results: the tensor core truncates its running sum at every step, an error that grows with k (measured 1.5e-6
// of the result at k = 2,048). They take k in chunks (p.chunk stages) into alternate accumulators, which the epilogue
// warps add in float32 registers (64 or 128 a thread); so does act'(), where it makes a float32 bias gradient. Measured
// error / time of 163,848 x 2,048 x 512 with a float32 residual: chunks of 512 4.7e-7 / 321 us, 768 6.8e-7 / 303, 1,024
// 1.0e-6 / 301.
//
// Bound, at 163,848 rows (times among other passes are up to 30 % longer: sw_power_cap at 1.2-1.5 GHz): k = 2,048 plain
// 254-262 us = 1.31-1.35 PFLOP/s (cuBLAS 253-275 on the same boxes), the MMAs; 512 x 2,048 plain 294 (cuBLAS 316-355);
// GELU 293-308 and e4m3 GELU 226, the latency of an epilogue chunk's steps (TMEM, arithmetic, shared memory, store), with no
// unit full (tensor pipe 57 and 35 %, issue slots 50 and 64 %); residual in float32 285-303, the MMAs and 8 bytes a value of
// HBM traffic; act'() with column sums at 81,924 rows 242, shared memory (x in, sums, result) and arithmetic. One product
// recomputed in the backward instead of keeping the pre-activation: 102 us of MMAs under that epilogue, against 8 bytes a
// value (0.2 ms) in float32. d_pre leaves in bf16, the operand of the two products that read it: 2.3e-3 of their results
// against 1.7e-3 for their own rounding alone; two bf16 parts of it would double both (81,924 rows: 2 x 120 us).
template <int TILE, bool X32, bool O32, bool PRE, bool SUM>
struct LinearCfg {
  static constexpr int CG = linear_pair(TILE) ? 2 : 1;
  static constexpr int BN = linear_tile_n(TILE);
  static constexpr int BNC = BN / CG;                    // rows of b per CTA
  static constexpr int A_BYTES = 128 * 128, B_BYTES = BNC * 128;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int EW = TILE == kTile256 ? 16 : 8;   // epilogue warps
  static constexpr int HC = BN / (EW / 4);               // columns of an epilogue warp
  static constexpr int CC = linear_chunk_cols(TILE, X32 || O32);
  static constexpr int NCH = HC / CC;
  static constexpr int X_ROW = CC * (X32 ? 4 : 2), O_ROW = CC * (O32 ? 4 : 2);  // bytes: 128 or 64
  static constexpr int SLOT = 32 * (X_ROW > O_ROW ? X_ROW : O_ROW);
  static constexpr int RED = 32 * 64;                    // PRE: 32 rows x 16 columns in float32, for the column sums
  static constexpr int NS = TILE == kTile256 ? (PRE ? 3 : 4) : TILE == kTile64 ? 6 : 5;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int THREADS = 128 + 32 * EW;
  // Registers at launch (65,536 over the threads, in steps of 8: 96 or 168) and after the warpgroups have traded: 128 x 40 +
  // 512 x 104 of 640 x 96, 128 x 56 + 256 x 224 = 384 x 168. Spilled: 104 to 224 bytes where k is added in chunks on
  // kTile256 (float32 results of odd widths, act'() with a float32 dy), at most 28 elsewhere.
  static constexpr int REGS_LOW = TILE == kTile256 ? 40 : 56, REGS_HIGH = TILE == kTile256 ? 104 : 224;
  static_assert(128 * REGS_LOW + 32 * EW * REGS_HIGH <= THREADS * (65536 / THREADS / 8 * 8), "more than the launch has");
  static constexpr int N_BAR = 2 * NS + 4 + 1 + EW;
  static constexpr int OFF_SLOT = NS * STAGE;            // per epilogue warp
  static constexpr int OFF_RED = OFF_SLOT + EW * SLOT;
  static constexpr int OFF_VEC = OFF_RED + (PRE ? EW * RED : 0);  // per epilogue warp: HC biases and HC scales
  static constexpr int OFF_BAR = OFF_VEC + EW * 2 * HC * 4;
  static constexpr int SMEM = OFF_BAR + N_BAR * 8 + 16 + 1024;
  static_assert(OFF_SLOT % 1024 == 0 && SLOT % 1024 == 0 && OFF_RED % 1024 == 0, "swizzle atoms");
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

// Offset of 16-byte piece i of row r in a chunk of ROW-byte rows (128-byte or 64-byte swizzle), and of one byte in it.
template <int ROW>
__device__ __forceinline__ uint32_t piece_at(int r, int i) {
  if constexpr (ROW == 128) return sw128_offset(r, i);
  return sw64_offset(r, i);
}
template <int ROW>
__device__ __forceinline__ uint32_t byte_at(int r, int b) { return piece_at<ROW>(r, b >> 4) + (b & 15); }
// The tiles of a CTA (pair), n fastest, then m, then the splits of k; the step's parts come from the host, so that the
// walk divides once (a division of 64 bits per tile held the MMA warp for 1,000 cycles).
struct TileWalk {
  int t, nt, mt, sp;
  __device__ __forceinline__ TileWalk(const LinearParams& p, int first) : t(first) {
    nt = first % p.n_tiles;
    const int r = first / p.n_tiles;
    mt = r % p.m_tiles;
    sp = r / p.m_tiles;
  }
  __device__ __forceinline__ void next(const LinearParams& p, int step) {
    t += step;
    nt += p.step_n;
    mt += p.step_m;
    sp += p.step_s;
    if (nt >= p.n_tiles) {
      nt -= p.n_tiles;
      ++mt;
    }
    if (mt >= p.m_tiles) {
      mt -= p.m_tiles;
      ++sp;
    }
  }
  __device__ __forceinline__ int kb0(const LinearParams& p) const { return sp * p.kb_q + min(sp, p.kb_r); }
  __device__ __forceinline__ int kb1(const LinearParams& p) const { return kb0(p) + p.kb_q + (sp < p.kb_r ? 1 : 0); }
};

__device__ __forceinline__ void st_shared_u16(uint32_t a, uint16_t v) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"(v) : "memory");
}
__device__ __forceinline__ void st_shared_u32(uint32_t a, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ uint16_t ld_shared_u16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
  return v;
}

template <int TILE, int ACT, bool X32, bool O32, bool PRE, bool SUM>
__global__ void __launch_bounds__(LinearCfg<TILE, X32, O32, PRE, SUM>::THREADS, 1)
    linear_tile_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                       const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_o,
                       const LinearParams p) {
  using C = LinearCfg<TILE, X32, O32, PRE, SUM>;
  constexpr int CG = C::CG;
  extern __shared__ uint8_t smem_linear[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_linear) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + C::OFF_BAR;
  auto a_st = [&](int s) { return sbase + s * C::STAGE; };
  auto b_st = [&](int s) { return sbase + s * C::STAGE + C::A_BYTES; };
  auto full = [&](int s) { return bar0 + 8 * s; };
  auto empty = [&](int s) { return bar0 + 8 * (C::NS + s); };
  auto acc_full = [&](int b) { return bar0 + 8 * (2 * C::NS + b); };
  auto acc_empty = [&](int b) { return bar0 + 8 * (2 * C::NS + 2 + b); };
  const uint32_t drain = bar0 + 8 * (2 * C::NS + 4);
  auto x_bar = [&](int w) { return bar0 + 8 * (2 * C::NS + 5 + w); };
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::OFF_BAR + C::N_BAR * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_BAR + C::N_BAR * 8 + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CG == 2 ? static_cast<int>(cluster_rank()) : 0;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::NS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), C::EW * CG);
    }
    mbar_init(drain, 1);
    for (int w = 0; w < C::EW; ++w) mbar_init(x_bar(w), 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_b);
    if (!p.out_direct) tma_prefetch_desc(&tm_o);
    if (p.x != nullptr && !p.x_direct) tma_prefetch_desc(&tm_x);
  }
  if (warp == 1) tmem_alloc_cg<CG>(smem_u32(tmem_holder), C::TMEM_COLS);
  tc_fence_before();
  __syncwarp();
  if constexpr (CG == 2) cluster_sync_all(); else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const int bk = p.fp8 ? 128 : 64;

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_LOW));
  if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------------ TMA producers (a: warp 0, b: warp 2)
    // CG = 2: both CTAs' bytes count on the first CTA's barrier, whose warp 0 expects them.
    const bool is_a = warp == 0;
    const bool mn = is_a ? p.a_mn : p.b_mn;
    const CUtensorMap* tm = is_a ? &tm_a : &tm_b;
    const int base = is_a ? rank * 128 : rank * C::BNC, boxes = is_a ? 2 : C::BNC / 64;
    uint32_t g = 0;
    bool ok = true;
    for (TileWalk w(p, first); w.t < p.items && ok; w.next(p, step)) {
      const int at = (is_a ? w.mt * 128 * CG : w.nt * C::BN) + base;
      const int kb1 = w.kb1(p);
      for (int kb = w.kb0(p); kb < kb1; ++kb, ++g) {
        const int st = g % C::NS;
        if (!(ok = poll_wait(empty(st), ((g / C::NS) & 1) ^ 1, abort_flag))) break;
        const uint32_t bar = CG == 2 ? map_to(full(st), 0) : full(st);
        const uint32_t dst = is_a ? a_st(st) : b_st(st);
        if (elect_one_sync()) {
          if (is_a && rank == 0) mbar_arrive_expect_tx(full(st), CG * C::STAGE);
          if (mn) {
            for (int i = 0; i < boxes; ++i) tile_load<CG>(dst + i * 8192, tm, at + 64 * i, kb * bk, bar);
          } else {
            tile_load<CG>(dst, tm, kb * bk, at, bar);
          }
        }
        __syncwarp();
      }
    }
    // Every stage used is consumed before this CTA may leave (CG = 2: its pair's MMAs read its stages, and arrive here).
    volatile int never = 0;
    if (ok) {
      for (uint32_t i = (g >= C::NS ? g - C::NS : 0); i < g; ++i) {
        if (!warp_wait(empty(i % C::NS), (i / C::NS) & 1, abort_flag)) break;
      }
    } else if (rank == 0) {
      // Gave up: the copies in flight land before TMEM and shared memory are released (bounded, abort flag ignored).
      for (uint32_t i = (g >= C::NS ? g - C::NS : 0); i < g; ++i) mbar_wait(full(i % C::NS), (i / C::NS) & 1, &never);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (rank == 0) {
      // float32 accumulation; operand format bf16 (1) or e4m3 (0); orders; N / 8; M / 16.
      const uint32_t idesc = (1u << 4) | (p.fp8 ? 0u : (1u << 7) | (1u << 10)) | (p.a_mn ? 1u << 15 : 0u) |
                             (p.b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(C::BN >> 3) << 17) |
                             (static_cast<uint32_t>(128 * CG >> 4) << 24);
      // Bytes between an operand's consecutive k steps (16 bf16 or 32 e4m3): along its 128-byte rows, or 16 rows.
      const uint32_t ka = (p.a_mn ? 2048u : 32u) >> 4, kbs = (p.b_mn ? 2048u : 32u) >> 4;
      const uint32_t a_lbo = p.a_mn ? 8192 : 16, b_lbo = p.b_mn ? 8192 : 16;
      uint32_t g = 0, acc_i = 0;
      bool ok = true;
      for (TileWalk w(p, first); w.t < p.items && ok; w.next(p, step)) {
        const int kb0 = w.kb0(p), kb1 = w.kb1(p);
        int buf = 0, left = 0;  // stages until the accumulator is handed over
        uint32_t d = 0;
        for (int kb = kb0; kb < kb1; ++kb, ++g) {
          const bool begin = left == 0;
          if (begin) {
            left = SUM ? min(p.chunk, kb1 - kb) : kb1 - kb;
            buf = acc_i & 1;
            if (!(ok = poll_wait(acc_empty(buf), ((acc_i >> 1) & 1) ^ 1, abort_flag))) break;
            tc_fence_after();
            d = tmem + buf * C::BN;
            ++acc_i;
          }
          --left;
          const int st = g % C::NS;
          if (!(ok = poll_wait(full(st), (g / C::NS) & 1, abort_flag))) break;
          tc_fence_after();
          const uint64_t ad = smem_desc(a_st(st), a_lbo, 1024), bd = smem_desc(b_st(st), b_lbo, 1024);
          if (elect_one_sync()) {
            if (p.fp8) {
#pragma unroll
              for (int i = 0; i < 4; ++i) mma<CG, true>(d, ad + 2 * i, bd + 2 * i, idesc, (!begin || i > 0) ? 1u : 0u);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                mma<CG, false>(d, ad + i * ka, bd + i * kbs, idesc, (!begin || i > 0) ? 1u : 0u);
            }
            commit<CG>(empty(st));
            if (left == 0) commit<CG>(acc_full(buf));
          }
          __syncwarp();
        }
      }
      if (elect_one_sync()) {
        if constexpr (CG == 2)
          asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(drain) : "memory");
        else
          mma_commit(drain);
      }
      __syncwarp();
      volatile int never = 0;
      mbar_wait(drain, 0, &never);
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_HIGH));
    // ------------------------------------------------------------------ epilogue
    const int ew = warp - 4, quarter = warp & 3, part = ew >> 2;
    constexpr int CC = C::CC;
    const uint32_t trow = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + part * C::HC;
    const uint32_t slot = sbase + C::OFF_SLOT + ew * C::SLOT;
    float* vec = reinterpret_cast<float*>(smem + C::OFF_VEC) + ew * 2 * C::HC;
    const uint32_t vec_s = smem_u32(vec);
    const bool has_x = p.x != nullptr;
    const bool x_tma = has_x && !p.x_direct;
    // One lane issues all of a warp's copies (elect.sync: from uniform registers), so its waits cover its stores.
    auto issue_x = [&](const TileWalk& w, int ch) {  // the residual (dy) of chunk ch of a tile into the slot
      mbar_arrive_expect_tx(x_bar(ew), 32 * C::X_ROW);
      tile_load<1>(slot, &tm_x, w.nt * C::BN + part * C::HC + ch * CC, w.mt * 128 * CG + rank * 128 + quarter * 32, x_bar(ew));
    };
    // Biases and scales of this warp's columns of a tile, HC / 32 a lane, read a tile ahead.
    float next_bias[C::HC / 32], next_scale[C::HC / 32];
    auto fetch_vec = [&](const TileWalk& w) {
#pragma unroll
      for (int i = 0; i < C::HC / 32; ++i) {
        const int c = w.nt * C::BN + part * C::HC + 32 * i + lane;
        next_bias[i] = 0.f;
        next_scale[i] = 1.f;
        if (w.t < p.items && c < p.n) {
          if (p.bias != nullptr)
            next_bias[i] = p.bias_bf16 ? __bfloat162float(static_cast<const bf16*>(p.bias)[c])
                                       : static_cast<const float*>(p.bias)[c];
          if (p.b_scale != nullptr) next_scale[i] = p.b_scale[c];
        }
      }
    };
    auto release = [&](int buf) {  // this warp has read the accumulator: the MMAs may overwrite it
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_cluster(map_to(acc_empty(buf), 0)); else mbar_arrive(acc_empty(buf));
      }
    };
    float rs = 1.f;  // this row's scale
    // 32 accumulated values of this lane's row, from column `at` of the warp's: scales, bias, activation (its slope).
    auto finish32 = [&](float* v, int at) {
      if (p.b_scale != nullptr) {
        const float2 r2 = pair(rs);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 c = ld_shared_f32x4(vec_s + (C::HC + at + 4 * i) * 4);
          const float4 b = ld_shared_f32x4(vec_s + (at + 4 * i) * 4);
          const float2 lo = ffma2(make_float2(v[4 * i], v[4 * i + 1]), fmul2(r2, make_float2(c.x, c.y)), make_float2(b.x, b.y));
          const float2 hi = ffma2(make_float2(v[4 * i + 2], v[4 * i + 3]), fmul2(r2, make_float2(c.z, c.w)), make_float2(b.z, b.w));
          v[4 * i] = lo.x;
          v[4 * i + 1] = lo.y;
          v[4 * i + 2] = hi.x;
          v[4 * i + 3] = hi.y;
        }
      } else if (p.bias != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 b = ld_shared_f32x4(vec_s + (at + 4 * i) * 4);
          const float2 lo = fadd2(make_float2(v[4 * i], v[4 * i + 1]), make_float2(b.x, b.y));
          const float2 hi = fadd2(make_float2(v[4 * i + 2], v[4 * i + 3]), make_float2(b.z, b.w));
          v[4 * i] = lo.x;
          v[4 * i + 1] = lo.y;
          v[4 * i + 2] = hi.x;
          v[4 * i + 3] = hi.y;
        }
      }
      if constexpr (ACT != 0) {
        if constexpr (O32) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = activate<ACT>(v[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) activate4<ACT, PRE>(v + 4 * i);
        }
      }
    };
    auto free_slot = [&] {  // the slot's last store has read it
      if (!p.out_direct && elect_one_sync()) store_wait_read<0>();
      __syncwarp();
    };
    // Rows that TMA cannot address (x or the output): lane = column, so that a row's 32 values are one access; eight
    // rows in flight, one pointer a row.
    auto gather_x = [&](int64_t row0, int col) {
      using T = std::conditional_t<X32, uint32_t, uint16_t>;
      const T* src = static_cast<const T*>(p.x) + row0 * p.ldx + col + lane;
      const int rows = static_cast<int>(min(static_cast<int64_t>(32), p.m - row0));
      const bool in0 = col + lane < p.n, in1 = CC == 64 && col + 32 + lane < p.n;
#pragma unroll 1
      for (int r0 = 0; r0 < 32; r0 += 8) {
        T t[8][2];
#pragma unroll
        for (int r = 0; r < 8; ++r, src += p.ldx) {
          const bool in = r0 + r < rows;
          t[r][0] = in && in0 ? __ldg(src) : T(0);
          if (CC == 64) t[r][1] = in && in1 ? __ldg(src + 32) : T(0);
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const uint32_t at = slot + r0 * C::X_ROW + byte_at<C::X_ROW>(r, static_cast<int>(sizeof(T)) * lane);
          if constexpr (X32) {
            st_shared_u32(at, t[r][0]);
          } else {
            st_shared_u16(at, t[r][0]);
            if (CC == 64) st_shared_u16(at ^ 64u, t[r][1]);
          }
        }
      }
      __syncwarp();
    };
    auto scatter_out = [&](int64_t row0, int col) {
      using T = std::conditional_t<O32, uint32_t, uint16_t>;
      T* dst = static_cast<T*>(p.out) + row0 * p.ldo + col + lane;
      const int rows = static_cast<int>(min(static_cast<int64_t>(32), p.m - row0));
      const bool in0 = col + lane < p.n, in1 = CC == 64 && col + 32 + lane < p.n;
#pragma unroll 1
      for (int r0 = 0; r0 < rows; r0 += 8) {
        T t[8][2];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const uint32_t at = slot + r0 * C::O_ROW + byte_at<C::O_ROW>(r, static_cast<int>(sizeof(T)) * lane);
          if constexpr (O32) {
            t[r][0] = ld_shared_u32(at);
          } else {
            t[r][0] = ld_shared_u16(at);
            if (CC == 64) t[r][1] = ld_shared_u16(at ^ 64u);
          }
        }
#pragma unroll
        for (int r = 0; r < 8; ++r, dst += p.ldo) {
          const bool in = r0 + r < rows;
          if (in && in0) *dst = t[r][0];
          if (CC == 64 && in && in1) dst[32] = t[r][1];
        }
      }
    };
    auto combine = [&](float& v, float x) { v = PRE ? v * x : v + x; };  // dy times the slope; the residual is added
    TileWalk w(p, first);
    if (x_tma && elect_one_sync()) issue_x(w, 0);
    __syncwarp();
    fetch_vec(w);
    uint32_t q = 0, acc_i = 0;
    bool ok = true;
    while (w.t < p.items) {
      TileWalk after = w;
      after.next(p, step);
      const int64_t row0 = static_cast<int64_t>(w.mt) * 128 * CG + rank * 128 + quarter * 32;
      const int col0 = w.nt * C::BN + part * C::HC;
      __syncwarp();  // the previous tile's reads of vec
#pragma unroll
      for (int i = 0; i < C::HC / 32; ++i) {
        vec[32 * i + lane] = next_bias[i];
        vec[C::HC + 32 * i + lane] = next_scale[i];
      }
      fetch_vec(after);
      rs = 1.f;
      if (p.a_scale != nullptr && row0 + lane < p.m) rs = p.a_scale[row0 + lane];
      __syncwarp();
      if (has_x && !x_tma) {  // the first chunk's x while the MMAs run
        free_slot();
        gather_x(row0, col0);
      }
      int buf = acc_i & 1;
      float sum[SUM ? C::HC : 1];
      if constexpr (SUM) {
#pragma unroll
        for (int i = 0; i < C::HC; ++i) sum[i] = 0.f;
        const int kb1 = w.kb1(p);
        for (int kb = w.kb0(p); kb < kb1; kb += p.chunk, ++acc_i) {
          buf = acc_i & 1;
          if (!(ok = warp_wait(acc_full(buf), (acc_i >> 1) & 1, abort_flag))) goto done;
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < C::HC; j += 16) {
            float u[16];
            tmem_ld16(trow + buf * C::BN + j, u);
            tmem_wait_ld();
            reg_fence(u);
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[j + i] += u[i];
          }
          release(buf);
        }
      } else {
        if (!(ok = warp_wait(acc_full(buf), (acc_i >> 1) & 1, abort_flag))) goto done;
        tc_fence_after();
        ++acc_i;
      }
#pragma unroll
      for (int ch = 0; ch < C::NCH; ++ch, ++q) {
        const int col = col0 + CC * ch;
        if (x_tma) {
          if (!(ok = warp_wait(x_bar(ew), q & 1, abort_flag))) goto done;
        } else if (ch > 0 || !has_x) {
          free_slot();
          if (has_x) gather_x(row0, col);
        }
#pragma unroll
        for (int h = 0; h < CC; h += 32) {
          float acc[32];
          float* v = acc;
          if constexpr (SUM) {
            v = sum + (SUM ? CC * ch + h : 0);
          } else {
            tmem_ld32(trow + buf * C::BN + CC * ch + h, acc);
            tmem_wait_ld();
            reg_fence(acc);
            if (ch == C::NCH - 1 && h == CC - 32) release(buf);
          }
          finish32(v, CC * ch + h);
          if (has_x) {
            if constexpr (X32) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 f = ld_shared_f32x4(slot + piece_at<C::X_ROW>(lane, i));
                combine(v[4 * i], f.x);
                combine(v[4 * i + 1], f.y);
                combine(v[4 * i + 2], f.z);
                combine(v[4 * i + 3], f.w);
              }
              if constexpr (!O32) __syncwarp();  // the result's rows are shorter than x's: every lane has read its own
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint4 u = ld_shared_u32x4(slot + piece_at<C::X_ROW>(lane, h / 8 + i));
                const uint32_t t[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  combine(v[8 * i + 2 * e], __uint_as_float(t[e] << 16));
                  combine(v[8 * i + 2 * e + 1], __uint_as_float(t[e] & 0xFFFF0000u));
                }
              }
            }
          }
          if constexpr (PRE) {
            if (p.colsum != nullptr) {
              // Column sums of the 32 rows in float32, across lanes, 16 columns at a time through shared memory: lane l
              // adds rows 4 (l / 4) + [0, 4) of columns 4 (l % 4) + [0, 4), and three exchanges join the eight groups
              // of rows, the first two of which also share out the columns. Rows past m have dy = 0.
              const uint32_t red = sbase + C::OFF_RED + ew * C::RED;
#pragma unroll
              for (int j = 0; j < 32; j += 16) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  st_shared_v4(red + sw64_offset(lane, i), __float_as_uint(v[j + 4 * i]), __float_as_uint(v[j + 4 * i + 1]),
                               __float_as_uint(v[j + 4 * i + 2]), __float_as_uint(v[j + 4 * i + 3]));
                __syncwarp();
                float2 c0 = make_float2(0.f, 0.f), c1 = c0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float4 f = ld_shared_f32x4(red + sw64_offset((lane & 28) + i, lane & 3));
                  c0 = fadd2(c0, make_float2(f.x, f.y));
                  c1 = fadd2(c1, make_float2(f.z, f.w));
                }
                const bool up = lane & 4, odd = lane & 8;
                const float2 send = up ? c0 : c1;
                float2 keep = up ? c1 : c0;
                keep.x += __shfl_xor_sync(0xffffffffu, send.x, 4);
                keep.y += __shfl_xor_sync(0xffffffffu, send.y, 4);
                float c = odd ? keep.y : keep.x;
                c += __shfl_xor_sync(0xffffffffu, odd ? keep.x : keep.y, 8);
                c += __shfl_xor_sync(0xffffffffu, c, 16);
                const int cc = col + h + j + 4 * (lane & 3) + 2 * up + odd;
                if (lane < 16 && row0 < p.m && cc < p.n) p.colsum[(row0 >> 5) * p.n + cc] = c;
              }
            }
          }
          if constexpr (O32) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              st_shared_v4(slot + piece_at<C::O_ROW>(lane, i), __float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                           __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              st_shared_v4(slot + piece_at<C::O_ROW>(lane, h / 8 + i), pack_bf16(v[8 * i], v[8 * i + 1]),
                           pack_bf16(v[8 * i + 2], v[8 * i + 3]), pack_bf16(v[8 * i + 4], v[8 * i + 5]),
                           pack_bf16(v[8 * i + 6], v[8 * i + 7]));
          }
        }
        if (p.out_direct) {
          __syncwarp();
          scatter_out(row0, col);
        }
        // The slot's writes before the store that reads them, its reads before the copy that overwrites them (without
        // the proxy fence loads were still on their way when the next chunk landed).
        fence_proxy_async_smem();
        __syncwarp();
        if (elect_one_sync()) {
          if (!p.out_direct) {
            if (row0 < p.m && col < p.n)
              tile_store(&tm_o, col, static_cast<int>(row0 + w.sp * p.split_rows), slot);
            store_commit();
          }
          if (x_tma && (ch + 1 < C::NCH || after.t < p.items)) {
            if (!p.out_direct) store_wait_read<0>();
            if (ch + 1 < C::NCH) issue_x(w, ch + 1); else issue_x(after, 0);
          }
        }
        __syncwarp();
      }
      w = after;
    }
  done:
    if (elect_one_sync()) store_wait_all();
    __syncwarp();
    if (!ok && x_tma) {
      // Gave up with a copy in flight: wait (bounded, abort flag ignored) until it has landed.
      volatile int never = 0;
      mbar_wait(x_bar(ew), q & 1, &never);
    }
  }
  tc_fence_before();
  __syncwarp();
  if constexpr (CG == 2) cluster_sync_all(); else __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc_cg<CG>(tmem, C::TMEM_COLS);
}

template <int TILE, int ACT, bool X32, bool O32, bool PRE, bool SUM>
cudaError_t launch_tile(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tx, const CUtensorMap& to,
                        const LinearParams& given, int sms, cudaStream_t stream) {
  LinearParams p = given;
  using C = LinearCfg<TILE, X32, O32, PRE, SUM>;
  auto kernel = linear_tile_kernel<TILE, ACT, X32, O32, PRE, SUM>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  const int groups = std::min(p.items, sms / C::CG);
  p.kb_q = p.k_blocks / p.splits;
  p.kb_r = p.k_blocks % p.splits;
  p.step_n = groups % p.n_tiles;
  p.step_m = groups / p.n_tiles % p.m_tiles;
  p.step_s = groups / p.n_tiles / p.m_tiles;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(groups * C::CG);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C::CG;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, ta, tb, tx, to, p);
}

template <int TILE, bool X32, bool O32, bool PRE, bool SUM>
cudaError_t by_act(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tx, const CUtensorMap& to,
                   const LinearParams& p, int sms, cudaStream_t st) {
  if (p.act == 1) return launch_tile<TILE, 1, X32, O32, PRE, SUM>(ta, tb, tx, to, p, sms, st);
  if (p.act == 2) return launch_tile<TILE, 2, X32, O32, PRE, SUM>(ta, tb, tx, to, p, sms, st);
  if constexpr (PRE)
    return cudaErrorInvalidValue;  // without an activation the gradient needs no product
  else
    return launch_tile<TILE, 0, X32, O32, PRE, SUM>(ta, tb, tx, to, p, sms, st);
}

template <int TILE>
cudaError_t by_type(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tx, const CUtensorMap& to,
                    const LinearParams& p, int sms, cudaStream_t st) {
  const bool sum = (p.k_blocks + p.splits - 1) / p.splits > p.chunk;  // more than one chunk of k: added in registers
  if (p.pre_grad) {
    if (sum)
      return p.x_f32 ? by_act<TILE, true, false, true, true>(ta, tb, tx, to, p, sms, st)
                     : by_act<TILE, false, false, true, true>(ta, tb, tx, to, p, sms, st);
    return p.x_f32 ? by_act<TILE, true, false, true, false>(ta, tb, tx, to, p, sms, st)
                   : by_act<TILE, false, false, true, false>(ta, tb, tx, to, p, sms, st);
  }
  if (!p.out_f32) return by_act<TILE, false, false, false, false>(ta, tb, tx, to, p, sms, st);
  return sum ? by_act<TILE, true, true, false, true>(ta, tb, tx, to, p, sms, st)
                                                          : by_act<TILE, true, true, false, false>(ta, tb, tx, to, p, sms, st);
}

// ---- the sum of a split product's parts, with the epilogue ----------------------------------------------------------

__device__ __forceinline__ float activate_any(int act, float x) {
  return act == 1 ? activate<1>(x) : act == 2 ? activate<2>(x) : x;
}
// acc at (row, col) through scales, bias, activation and residual, to out.
__device__ __forceinline__ void finish(const LinearParams& p, int64_t row, int col, float acc) {
  if (p.b_scale != nullptr) acc *= p.a_scale[row] * p.b_scale[col];
  if (p.bias != nullptr)
    acc += p.bias_bf16 ? __bfloat162float(static_cast<const bf16*>(p.bias)[col]) : static_cast<const float*>(p.bias)[col];
  acc = activate_any(p.act, acc);
  if (p.x != nullptr) {
    const int64_t at = row * p.ldx + col;
    acc += p.x_f32 ? static_cast<const float*>(p.x)[at] : __bfloat162float(static_cast<const bf16*>(p.x)[at]);
  }
  if (p.out_f32)
    static_cast<float*>(p.out)[row * p.ldo + col] = acc;
  else
    static_cast<bf16*>(p.out)[row * p.ldo + col] = __float2bfloat16_rn(acc);
}

// One column per thread, a row per block row: the parts (in L2, just written) are read once, in split order.
__global__ void __launch_bounds__(256) linear_split_sum_kernel(const float* __restrict__ part, int64_t ldp,
                                                               const LinearParams p) {
  const int64_t row = blockIdx.x;
  const int col = blockIdx.y * 256 + threadIdx.x;
  if (col >= p.n) return;
  float acc = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) acc += part[(s * p.split_rows + row) * ldp + col];
  finish(p, row, col, acc);
}

// ---- few rows ------------------------------------------------------------------------------------------------------

// m <= M rows of a against b [n, k]: a warp per output column, lanes along k, so that b, which is nearly all there is to
// read, streams through wide coalesced loads and a comes from L1. Sums in float32, joined by shuffles.
template <int M, bool FP8, bool WIDE>
__global__ void __launch_bounds__(128) linear_rows_kernel(const uint8_t* __restrict__ a, int64_t lda,
                                                          const uint8_t* __restrict__ b, int64_t ldb,
                                                          const LinearParams p) {
  constexpr int ES = FP8 ? 1 : 2;
  constexpr int V = WIDE ? 16 / ES : 1;
  const int col = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (col >= p.n) return;  // whole warps
  auto widen = [](const uint8_t* src, float (&v)[V]) {
    if constexpr (WIDE) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(src));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (FP8) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t f16x2;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f16x2) : "h"(static_cast<uint16_t>(w[i] >> (16 * h))));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&f16x2));
            v[4 * i + 2 * h] = f.x;
            v[4 * i + 2 * h + 1] = f.y;
          }
        } else {
          const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
          v[2 * i] = f.x;
          v[2 * i + 1] = f.y;
        }
      }
    } else if constexpr (FP8) {
      uint32_t f16x2;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f16x2) : "h"(static_cast<uint16_t>(__ldg(src))));
      v[0] = __half22float2(*reinterpret_cast<const __half2*>(&f16x2)).x;
    } else {
      v[0] = __bfloat162float(*reinterpret_cast<const bf16*>(src));
    }
  };
  float acc[M];
#pragma unroll
  for (int r = 0; r < M; ++r) acc[r] = 0.f;
  const uint8_t* brow = b + static_cast<int64_t>(col) * ldb * ES;
#pragma unroll 4
  for (int at = lane * V; at < p.k; at += 32 * V) {
    float w[V];
    widen(brow + static_cast<int64_t>(at) * ES, w);
#pragma unroll
    for (int r = 0; r < M; ++r) {
      if (r < p.m) {
        float x[V];
        widen(a + (r * lda + at) * ES, x);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[r] = fmaf(x[e], w[e], acc[r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < M; ++r)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
#pragma unroll
  for (int r = 0; r < M; ++r)
    if (lane == r && r < p.m) finish(p, r, col, acc[r]);
}

template <int M, bool FP8, bool WIDE>
cudaError_t rows_go(const void* a, int64_t lda, const void* b, int64_t ldb, const LinearParams& p, cudaStream_t st) {
  linear_rows_kernel<M, FP8, WIDE><<<(p.n + 3) / 4, 128, 0, st>>>(static_cast<const uint8_t*>(a), lda,
                                                                  static_cast<const uint8_t*>(b), ldb, p);
  return cudaGetLastError();
}
template <int M>
cudaError_t rows_by_type(const void* a, int64_t lda, const void* b, int64_t ldb, bool wide, const LinearParams& p,
                         cudaStream_t st) {
  if (p.fp8) return wide ? rows_go<M, true, true>(a, lda, b, ldb, p, st) : rows_go<M, true, false>(a, lda, b, ldb, p, st);
  return wide ? rows_go<M, false, true>(a, lda, b, ldb, p, st) : rows_go<M, false, false>(a, lda, b, ldb, p, st);
}

// ---- packing and the gradient without an activation ----------------------------------------------------------------

// Rows of any stride and base to rows of whole 16 bytes: a warp per row, a lane gathers 16 bytes and stores them at once
// (the last piece filled up with zeros).
template <class T>
__global__ void __launch_bounds__(256) pack_rows_kernel(const T* __restrict__ src, int64_t lds, T* __restrict__ dst,
                                                        int64_t ldd, int64_t rows, int64_t cols) {
  constexpr int V = 16 / sizeof(T);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const T* from = src + row * lds;
#pragma unroll 2
  for (int64_t j = (threadIdx.x & 31) * V; j < cols; j += 32 * V) {
    __align__(16) T v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = j + e < cols ? from[j + e] : T(0);
    *reinterpret_cast<uint4*>(dst + row * ldd + j) = *reinterpret_cast<const uint4*>(v);
  }
}

// A block takes 32 V columns (lane = V columns) and every gridDim.y-th group of eight rows; partial sums per block in
// float32, added over its eight warps in order.
template <bool X32, int V>
__global__ void __launch_bounds__(256) grad_cast_kernel(const void* __restrict__ x, int64_t ldx, int64_t m, int n,
                                                        bf16* __restrict__ cast, int64_t ldc, float* __restrict__ part) {
  __shared__ float red[8][32 * V + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (blockIdx.x * 32 + lane) * V;
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = 0.f;
  if (col < n) {
#pragma unroll 4
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * 8 + warp; r < m; r += static_cast<int64_t>(gridDim.y) * 8) {
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
            const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
          }
        }
      } else {
        v[0] = X32 ? static_cast<const float*>(x)[r * ldx + col]
                   : __bfloat162float(static_cast<const bf16*>(x)[r * ldx + col]);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] += v[e];
      if (cast != nullptr) {
        if constexpr (V == 8) {
          uint4 u;
          u.x = pack_bf16(v[0], v[1]);
          u.y = pack_bf16(v[2], v[3]);
          u.z = pack_bf16(v[4], v[5]);
          u.w = pack_bf16(v[6], v[7]);
          *reinterpret_cast<uint4*>(cast + r * ldc + col) = u;
        } else {
          cast[r * ldc + col] = __float2bfloat16_rn(v[0]);
        }
      }
    }
  }
  if (part == nullptr) return;
#pragma unroll
  for (int e = 0; e < V; ++e) red[warp][lane * V + e] = s[e];
  __syncthreads();
  for (int j = threadIdx.x; j < 32 * V; j += 256) {
    const int c = blockIdx.x * 32 * V + j;
    if (c < n) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) t += red[w][j];
      part[static_cast<int64_t>(blockIdx.y) * n + c] = t;
    }
  }
}

}  // namespace

cudaError_t launch_linear_tiles(int tile, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tx,
                                const CUtensorMap& to, const LinearParams& p, int sms, cudaStream_t st) {
  if (tile == kTile256) return by_type<kTile256>(ta, tb, tx, to, p, sms, st);
  if (tile == kTile256Long) return by_type<kTile256Long>(ta, tb, tx, to, p, sms, st);
  if (tile == kTile128) return by_type<kTile128>(ta, tb, tx, to, p, sms, st);
  return by_type<kTile64>(ta, tb, tx, to, p, sms, st);
}

cudaError_t launch_linear_split_sum(const float* part, int64_t ldp, const LinearParams& p, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.m), static_cast<unsigned>((p.n + 255) / 256));
  linear_split_sum_kernel<<<grid, 256, 0, st>>>(part, ldp, p);
  return cudaGetLastError();
}

cudaError_t launch_linear_rows(const void* a, int64_t lda, const void* b, int64_t ldb, bool wide, const LinearParams& p,
                               cudaStream_t st) {
  if (p.m <= 1) return rows_by_type<1>(a, lda, b, ldb, wide, p, st);
  if (p.m <= 2) return rows_by_type<2>(a, lda, b, ldb, wide, p, st);
  if (p.m <= 4) return rows_by_type<4>(a, lda, b, ldb, wide, p, st);
  return rows_by_type<kLinearRowsMax>(a, lda, b, ldb, wide, p, st);
}

cudaError_t launch_pack_rows(const void* src, int64_t lds, void* dst, int64_t ldd, int64_t rows, int64_t cols, int es,
                             cudaStream_t st) {
  const int64_t blocks = (rows + 7) / 8;
  if (blocks == 0) return cudaSuccess;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  if (es == 1)
    pack_rows_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(static_cast<const uint8_t*>(src), lds,
                                                                    static_cast<uint8_t*>(dst), ldd, rows, cols);
  else
    pack_rows_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(static_cast<const uint16_t*>(src), lds,
                                                                    static_cast<uint16_t*>(dst), ldd, rows, cols);
  return cudaGetLastError();
}

int grad_cast_blocks(int64_t m, int n, int sms) {
  const int64_t across = (n + 255) / 256;
  const int64_t want = std::max<int64_t>(1, 8 * static_cast<int64_t>(sms) / across);
  return static_cast<int>(std::min<int64_t>(want, std::max<int64_t>(1, (m + 7) / 8)));
}

cudaError_t launch_grad_cast(const void* x, bool x_f32, int64_t ldx, int64_t m, int n, void* cast, int64_t ldc,
                             float* part, int blocks, bool wide, cudaStream_t st) {
  const int v = wide ? 8 : 1;
  const dim3 grid(static_cast<unsigned>((n + 32 * v - 1) / (32 * v)), static_cast<unsigned>(blocks));
  auto* c = static_cast<bf16*>(cast);
  if (x_f32) {
    if (wide) grad_cast_kernel<true, 8><<<grid, 256, 0, st>>>(x, ldx, m, n, c, ldc, part);
    else grad_cast_kernel<true, 1><<<grid, 256, 0, st>>>(x, ldx, m, n, c, ldc, part);
  } else {
    if (wide) grad_cast_kernel<false, 8><<<grid, 256, 0, st>>>(x, ldx, m, n, c, ldc, part);
    else grad_cast_kernel<false, 1><<<grid, 256, 0, st>>>(x, ldx, m, n, c, ldc, part);
  }
  return cudaGetLastError();
}

cudaError_t take_linear_error(unsigned int* word) {
  cudaError_t e = cudaMemcpyFromSymbol(word, g_device_error, sizeof(*word));
  if (e != cudaSuccess) return e;
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
}

}  // namespace fwn
