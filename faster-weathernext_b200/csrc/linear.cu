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
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
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

// -log2(e) times the logistic function's argument: GELU in its tanh form is x sigma(2 u), u = c0 (x + c1 x^3); swish is
// x sigma(x). Written through sigma both keep their relative precision where they are small.
template <int ACT>
__device__ __forceinline__ float neg_arg(float x) {
  if constexpr (ACT == 1) return (-2.f * kLog2e * kGeluC0) * fmaf(kGeluC1 * x, x * x, x);
  return -kLog2e * x;
}
template <int ACT>
__device__ __forceinline__ float activate(float x) {
  if constexpr (ACT == 0) return x;
  return x * rcp(1.f + ex2(neg_arg<ACT>(x)));
}
// d/dx: sigma + x sigma (1 - sigma) z', z' = 2 c0 (1 + 3 c1 x^2) or 1. x is clamped to where the slope has long reached
// 0 or 1, and the exponent below overflow, so that the products stay finite.
template <int ACT>
__device__ __forceinline__ float activate_grad(float x) {
  if constexpr (ACT == 0) return 1.f;
  constexpr float kMost = ACT == 1 ? 30.f : 100.f;
  const float xc = x != x ? x : fminf(fmaxf(x, -kMost), kMost);
  const float e = ex2(fminf(neg_arg<ACT>(xc), 100.f));
  const float s = rcp(1.f + e);
  const float z1 = ACT == 1 ? 2.f * kGeluC0 * fmaf(3.f * kGeluC1 * xc, xc, 1.f) : 1.f;
  const float r = fmaf(xc * s * z1, e * s, s);
  return x != x ? x : r;
}

// ---- tensor-core kernel --------------------------------------------------------------------------------------------

// Persistent; a CTA (CG = 1) or a pair of CTAs on two SMs (CG = 2) takes output tiles of 128 CG x BN, walked with n
// fastest so that the tiles in flight share their rows of a in L2. Warps:
//   0      TMA producer: 128 bytes of k (64 bf16, 128 e4m3) of 128 rows of a and of BN / CG rows of b per stage (with
//          m or n contiguous: 64 rows of k by 64 columns, one box per 64);
//   1      MMA issuer (CG = 2: of the pair's first CTA, for both), into one of two TMEM accumulators;
//   2-9    epilogue: warp w reads TMEM lanes 32 (w % 4) + [0, 32) (rows) and one half of the tile's columns, 32 at a
//          time; the residual (or dy) chunk of 32 x 32 arrives by TMA in a slot of the warp's own, the result replaces
//          it there and leaves by TMA, so that a tile's epilogue overlaps the next tile's MMAs.
// Ragged edges: TMA fills rows and columns past the tensors with zeros and clips stores. Why a pair on 256 x 256: per
// 64 of k an SM then takes in 32 KB for 512 cycles of MMA, half the L2 traffic per FLOP of 128 x 128 and two thirds of
// 128 x 256, which held that form at 1.14 PFLOP/s. The small tiles spread products of few rows over the SMs.
template <int TILE, bool F32>
struct LinearCfg {
  static constexpr int CG = TILE == kTile256 ? 2 : 1;
  static constexpr int BN = linear_tile_n(TILE);
  static constexpr int BNC = BN / CG;                    // rows of b per CTA
  static constexpr int A_BYTES = 128 * 128, B_BYTES = BNC * 128;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int HC = BN / 2, NCH = HC / 32;       // columns and chunks of an epilogue warp
  static constexpr int SLOT = F32 ? 4096 : 2048;         // one 32 x 32 chunk (float32 if x or the output is)
  static constexpr int NSLOT = F32 ? 2 : 3;
  static constexpr int NS = TILE == kTile64 ? 6 : F32 ? 4 : 5;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int THREADS = 320;
  static constexpr int N_BAR = 2 * NS + 4 + 1 + 8 * NSLOT;
  static constexpr int OFF_SLOT = NS * STAGE;
  static constexpr int OFF_VEC = OFF_SLOT + 8 * NSLOT * SLOT;  // per epilogue warp: HC biases and HC scales
  static constexpr int OFF_BAR = OFF_VEC + 8 * 2 * HC * 4;
  static constexpr int SMEM = OFF_BAR + N_BAR * 8 + 16 + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory budget");
};

// Offset of column c (0..31) of row r in a 32 x 32 chunk: rows of 64 (bf16, 64-byte swizzle) or 128 bytes (float32).
template <bool F32>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  if constexpr (F32) return sw128_offset(r, c >> 2) + ((c & 3) << 2);
  return sw64_offset(r, c >> 3) + ((c & 7) << 1);
}
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

template <int TILE, int ACT, bool X32, bool O32, bool PRE>
__global__ void __maxnreg__(168)
    linear_tile_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                       const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_o,
                       const LinearParams p) {
  using C = LinearCfg<TILE, X32 || O32>;
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
  auto slot_bar = [&](int w, int s) { return bar0 + 8 * (2 * C::NS + 5 + w * C::NSLOT + s); };
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
      mbar_init(acc_empty(b), 8 * CG);
    }
    mbar_init(drain, 1);
    for (int i = 0; i < 8 * C::NSLOT; ++i) mbar_init(slot_bar(0, i), 1);
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

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    // CG = 2: both CTAs' bytes count on the first CTA's barrier, whose producer expects them.
    uint32_t g = 0;
    bool ok = true;
    for (int t = first; t < p.items && ok; t += step) {
      const int split = t / (p.m_tiles * p.n_tiles), mn = t % (p.m_tiles * p.n_tiles);
      const int m0 = (mn / p.n_tiles) * 128 * CG + rank * 128, n0 = (mn % p.n_tiles) * C::BN + rank * C::BNC;
      const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * split / p.splits);
      const int kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (split + 1) / p.splits);
      for (int kb = kb0; kb < kb1; ++kb, ++g) {
        const int st = g % C::NS;
        if (!(ok = mbar_wait(empty(st), ((g / C::NS) & 1) ^ 1, abort_flag))) break;
        if (lane == 0) {
          if (rank == 0) mbar_arrive_expect_tx(full(st), CG * C::STAGE);
          const uint32_t bar = CG == 2 ? map_to(full(st), 0) : full(st);
          if (p.a_mn) {
            for (int i = 0; i < 2; ++i) tile_load<CG>(a_st(st) + i * 8192, &tm_a, m0 + 64 * i, kb * bk, bar);
          } else {
            tile_load<CG>(a_st(st), &tm_a, kb * bk, m0, bar);
          }
          if (p.b_mn) {
            for (int i = 0; i < C::BNC / 64; ++i) tile_load<CG>(b_st(st) + i * 8192, &tm_b, n0 + 64 * i, kb * bk, bar);
          } else {
            tile_load<CG>(b_st(st), &tm_b, kb * bk, n0, bar);
          }
        }
        __syncwarp();
      }
    }
    // Every stage used is consumed before this CTA may leave (CG = 2: its pair's MMAs read its stages, and arrive here).
    volatile int never = 0;
    if (ok) {
      for (uint32_t i = (g >= C::NS ? g - C::NS : 0); i < g; ++i) {
        if (!mbar_wait(empty(i % C::NS), (i / C::NS) & 1, abort_flag)) break;
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
      for (int t = first; t < p.items && ok; t += step, ++acc_i) {
        const int split = t / (p.m_tiles * p.n_tiles);
        const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * split / p.splits);
        const int kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (split + 1) / p.splits);
        const int buf = acc_i & 1;
        if (!(ok = warp_wait(acc_empty(buf), ((acc_i >> 1) & 1) ^ 1, abort_flag))) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * C::BN;
        for (int kb = kb0; kb < kb1; ++kb, ++g) {
          const int st = g % C::NS;
          if (!(ok = warp_wait(full(st), (g / C::NS) & 1, abort_flag))) break;
          tc_fence_after();
          const uint64_t ad = smem_desc(a_st(st), a_lbo, 1024), bd = smem_desc(b_st(st), b_lbo, 1024);
          if (elect_one_sync()) {
            if (p.fp8) {
#pragma unroll
              for (int i = 0; i < 4; ++i) mma<CG, true>(d, ad + 2 * i, bd + 2 * i, idesc, (kb > kb0 || i > 0) ? 1u : 0u);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                mma<CG, false>(d, ad + i * ka, bd + i * kbs, idesc, (kb > kb0 || i > 0) ? 1u : 0u);
            }
            commit<CG>(empty(st));
            if (kb == kb1 - 1) commit<CG>(acc_full(buf));
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
  } else {
    // ------------------------------------------------------------------ epilogue
    const int ew = warp - 2, quarter = warp & 3, half = ew >> 2;
    const uint32_t trow = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * C::HC;
    const uint32_t slots = sbase + C::OFF_SLOT + ew * C::NSLOT * C::SLOT;
    float* vec = reinterpret_cast<float*>(smem + C::OFF_VEC) + ew * 2 * C::HC;
    const uint32_t vec_s = smem_u32(vec);
    const bool has_x = p.x != nullptr;
    const bool x_tma = has_x && !p.x_direct;
    const uint32_t my_items = p.items > first ? (p.items - first + step - 1) / step : 0;
    const uint32_t chunks = my_items * C::NCH;
    // First row and column of chunk q of this warp (its item's tile, the warp's half and quarter).
    auto place = [&](uint32_t q, int64_t& row, int& col) {
      const int t = first + static_cast<int>(q / C::NCH) * step;
      const int mn = t % (p.m_tiles * p.n_tiles);
      row = static_cast<int64_t>(mn / p.n_tiles) * 128 * CG + rank * 128 + quarter * 32;
      col = (mn % p.n_tiles) * C::BN + half * C::HC + static_cast<int>(q % C::NCH) * 32;
    };
    auto issue_x = [&](uint32_t q) {  // lane 0: chunk q's residual (dy) into its slot
      if (q >= chunks) return;
      int64_t row;
      int col;
      place(q, row, col);
      const int s = q % C::NSLOT;
      mbar_arrive_expect_tx(slot_bar(ew, s), 32 * 32 * (X32 ? 4 : 2));
      tile_load<1>(slots + s * C::SLOT, &tm_x, col, static_cast<int>(row), slot_bar(ew, s));
    };
    uint32_t issued = 0;
    if (x_tma) {
      if (lane == 0)
        for (int i = 0; i < C::NSLOT; ++i) issue_x(i);
      issued = C::NSLOT;
    }
    uint32_t q = 0, acc_i = 0;
    bool ok = true;
    for (int t = first; t < p.items && ok; t += step, ++acc_i) {
      const int split = t / (p.m_tiles * p.n_tiles), mn = t % (p.m_tiles * p.n_tiles);
      const int buf = acc_i & 1;
      const int64_t row0 = static_cast<int64_t>(mn / p.n_tiles) * 128 * CG + rank * 128 + quarter * 32;
      const int col0 = (mn % p.n_tiles) * C::BN + half * C::HC;
      __syncwarp();  // the previous tile's reads of vec
#pragma unroll
      for (int j = lane; j < C::HC; j += 32) {
        const int c = col0 + j;
        float b = 0.f, s = 1.f;
        if (c < p.n) {
          if (p.bias != nullptr)
            b = p.bias_bf16 ? __bfloat162float(static_cast<const bf16*>(p.bias)[c]) : static_cast<const float*>(p.bias)[c];
          if (p.b_scale != nullptr) s = p.b_scale[c];
        }
        vec[j] = b;
        vec[C::HC + j] = s;
      }
      float rs = 1.f;
      if (p.a_scale != nullptr && row0 + lane < p.m) rs = p.a_scale[row0 + lane];
      __syncwarp();
      if (!(ok = warp_wait(acc_full(buf), (acc_i >> 1) & 1, abort_flag))) break;
      tc_fence_after();
#pragma unroll 1
      for (int ch = 0; ch < C::NCH; ++ch, ++q) {
        const int s = q % C::NSLOT;
        const uint32_t slot = slots + s * C::SLOT;
        const int col = col0 + 32 * ch;
        float v[32];
        tmem_ld32(trow + buf * C::BN + 32 * ch, v);
        if (has_x) {
          if (x_tma) {
            if (!(ok = warp_wait(slot_bar(ew, s), (q / C::NSLOT) & 1, abort_flag))) break;
          } else {
            if (lane == 0) store_wait_read<C::NSLOT - 1>();
            __syncwarp();
            // Rows that TMA cannot address: lane = column, so that a row's 32 values are one access.
#pragma unroll 8
            for (int r = 0; r < 32; ++r) {
              const bool in = row0 + r < p.m && col + lane < p.n;
              const int64_t at = (row0 + r) * p.ldx + col + lane;
              if constexpr (X32)
                st_shared_u32(slot + chunk_at<true>(r, lane), in ? static_cast<const uint32_t*>(p.x)[at] : 0u);
              else
                st_shared_u16(slot + chunk_at<false>(r, lane), in ? static_cast<const uint16_t*>(p.x)[at] : uint16_t(0));
            }
            __syncwarp();
          }
        } else {
          if (lane == 0) store_wait_read<C::NSLOT - 1>();
          __syncwarp();
        }
        tmem_wait_ld();
        reg_fence(v);
        if (ch == C::NCH - 1) {
          // The accumulator has been read: the next tile but one may overwrite it.
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 2) mbar_arrive_cluster(map_to(acc_empty(buf), 0)); else mbar_arrive(acc_empty(buf));
          }
        }
        if (p.b_scale != nullptr) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 c = ld_shared_f32x4(vec_s + (C::HC + 32 * ch + 4 * i) * 4);
            v[4 * i] *= rs * c.x;
            v[4 * i + 1] *= rs * c.y;
            v[4 * i + 2] *= rs * c.z;
            v[4 * i + 3] *= rs * c.w;
          }
        }
        if (p.bias != nullptr) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float4 b = ld_shared_f32x4(vec_s + (32 * ch + 4 * i) * 4);
            v[4 * i] += b.x;
            v[4 * i + 1] += b.y;
            v[4 * i + 2] += b.z;
            v[4 * i + 3] += b.w;
          }
        }
        if constexpr (!PRE) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = activate<ACT>(v[i]);
        }
        // x: the residual is added; dy is multiplied by the activation's slope.
        if (has_x) {
          auto take = [&](int i, float x) { v[i] = PRE ? x * activate_grad<ACT>(v[i]) : v[i] + x; };
          if constexpr (X32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 f = ld_shared_f32x4(slot + sw128_offset(lane, i));
              take(4 * i, f.x);
              take(4 * i + 1, f.y);
              take(4 * i + 2, f.z);
              take(4 * i + 3, f.w);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4 u = ld_shared_u32x4(slot + sw64_offset(lane, i));
              const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]));
                take(8 * i + 2 * e, f.x);
                take(8 * i + 2 * e + 1, f.y);
              }
            }
          }
          __syncwarp();  // every lane has read the chunk before any writes it
        }
        if constexpr (PRE) {
          if (p.colsum != nullptr) {
            // Column sums of the 32 rows in float32: five exchanges that halve the columns a lane holds leave lane l
            // with column l. Rows past m have dy = 0.
            float c[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) c[i] = v[i];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                if (i < o) {
                  const bool up = (lane & o) != 0;
                  const float send = up ? c[i] : c[i + o], keep = up ? c[i + o] : c[i];
                  c[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
                }
              }
            }
            if (row0 < p.m && col + lane < p.n) p.colsum[(row0 >> 5) * p.n + col + lane] = c[0];
          }
        }
        if constexpr (O32) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            st_shared_v4(slot + sw128_offset(lane, i), __float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                         __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            st_shared_v4(slot + sw64_offset(lane, i), pack_bf16(v[8 * i], v[8 * i + 1]), pack_bf16(v[8 * i + 2], v[8 * i + 3]),
                         pack_bf16(v[8 * i + 4], v[8 * i + 5]), pack_bf16(v[8 * i + 6], v[8 * i + 7]));
        }
        if (p.out_direct) {
          __syncwarp();
#pragma unroll 8
          for (int r = 0; r < 32; ++r) {
            if (row0 + r < p.m && col + lane < p.n) {
              const int64_t at = (row0 + r) * p.ldo + col + lane;
              if constexpr (O32)
                static_cast<uint32_t*>(p.out)[at] = ld_shared_u32(slot + chunk_at<true>(r, lane));
              else
                static_cast<uint16_t*>(p.out)[at] = ld_shared_u16(slot + chunk_at<false>(r, lane));
            }
          }
          fence_proxy_async_smem();  // these reads before the slot's next TMA load
          __syncwarp();
          if (x_tma && lane == 0) issue_x(issued);
          ++issued;
        } else {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (row0 < p.m && col < p.n)
              tile_store(&tm_o, col, static_cast<int>(row0 + split * p.split_rows), slot);
            store_commit();
            if (x_tma) {
              // The chunk before this one has left its slot: load into it.
              store_wait_read<1>();
              if (q > 0) issue_x(issued);
            }
          }
          if (q > 0) ++issued;
        }
      }
    }
    if (lane == 0) store_wait_all();
    if (!ok && x_tma && lane == 0) {
      // Gave up with copies in flight: wait (bounded, abort flag ignored) until they have landed.
      volatile int never = 0;
      for (uint32_t i = q; i < issued && i < chunks; ++i) mbar_wait(slot_bar(ew, i % C::NSLOT), (i / C::NSLOT) & 1, &never);
    }
  }
  tc_fence_before();
  __syncwarp();
  if constexpr (CG == 2) cluster_sync_all(); else __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc_cg<CG>(tmem, C::TMEM_COLS);
}

template <int TILE, int ACT, bool X32, bool O32, bool PRE>
cudaError_t launch_tile(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tx, const CUtensorMap& to,
                        const LinearParams& p, int sms, cudaStream_t stream) {
  using C = LinearCfg<TILE, X32 || O32>;
  auto kernel = linear_tile_kernel<TILE, ACT, X32, O32, PRE>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  const int groups = std::min(p.items, sms / C::CG);
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

template <int TILE, bool X32, bool O32, bool PRE>
cudaError_t by_act(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tx, const CUtensorMap& to,
                   const LinearParams& p, int sms, cudaStream_t st) {
  if (p.act == 1) return launch_tile<TILE, 1, X32, O32, PRE>(ta, tb, tx, to, p, sms, st);
  if (p.act == 2) return launch_tile<TILE, 2, X32, O32, PRE>(ta, tb, tx, to, p, sms, st);
  if constexpr (PRE)
    return cudaErrorInvalidValue;  // without an activation the gradient needs no product
  else
    return launch_tile<TILE, 0, X32, O32, PRE>(ta, tb, tx, to, p, sms, st);
}

template <int TILE>
cudaError_t by_type(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tx, const CUtensorMap& to,
                    const LinearParams& p, int sms, cudaStream_t st) {
  if (p.pre_grad)
    return p.x_f32 ? by_act<TILE, true, false, true>(ta, tb, tx, to, p, sms, st)
                   : by_act<TILE, false, false, true>(ta, tb, tx, to, p, sms, st);
  return p.out_f32 ? by_act<TILE, true, true, false>(ta, tb, tx, to, p, sms, st)
                   : by_act<TILE, false, false, false>(ta, tb, tx, to, p, sms, st);
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

template <class T>
__global__ void __launch_bounds__(256) pack_rows_kernel(const T* __restrict__ src, int64_t lds, T* __restrict__ dst,
                                                        int64_t ldd, int64_t rows, int64_t cols) {
  const int64_t per = (cols + 255) / 256;
  const int64_t row = blockIdx.x / per, col = (blockIdx.x % per) * 256 + threadIdx.x;
  if (row < rows && col < cols) dst[row * ldd + col] = src[row * lds + col];
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
  const int64_t blocks = rows * ((cols + 255) / 256);
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
