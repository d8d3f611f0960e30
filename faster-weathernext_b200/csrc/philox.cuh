// Dropout's random numbers: Philox4x32-10, the counter-based generator of Salmon, Moraes, Dror and Shaw ("Parallel random
// numbers: as easy as 1, 2, 3", SC 2011). A mask is a function of the value's place in its tensor, so forward and backward
// compute it again instead of keeping it, whatever their tiles, strides or launch shapes.
//
// Value i takes the 16-bit number i % 8 (the words' low halves first) of the counter (i / 8, site, 0) under the 64-bit key
// `seed`, and is dropped where that is below `threshold`. Sixteen bits: one call of the generator, some 80 integer
// instructions, serves the eight values of a thread's access (with 32 bits a value the generator alone would take 50 us at
// 163,848 x 512, as long as the memory traffic of half a dropout pass); the probability is a multiple of 2^-16, and the factor of what is kept is that
// probability's own.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace fwn {

struct DropParams {
  const unsigned long long* seed_at;  // the seed on the device, or null: `seed`
  unsigned long long seed;
  uint32_t site, threshold;           // of 65,536; 0: nothing is dropped
  float factor;                       // 65536 / (65536 - threshold); 0 at 65,536
};

inline DropParams drop_params(uint64_t seed, const void* seed_at, uint32_t site, uint32_t threshold) {
  return {static_cast<const unsigned long long*>(seed_at), seed, site, threshold,
          threshold < 65536u ? 65536.f / static_cast<float>(65536u - threshold) : 0.f};
}

__device__ __forceinline__ uint4 philox(uint64_t counter, uint32_t site, uint64_t seed) {
  uint32_t c0 = static_cast<uint32_t>(counter), c1 = static_cast<uint32_t>(counter >> 32), c2 = site, c3 = 0;
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(0xD2511F53u) * c0, p1 = static_cast<uint64_t>(0xCD9E8D57u) * c2;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(p1);
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint64_t drop_seed(const DropParams& p) { return p.seed_at != nullptr ? __ldg(p.seed_at) : p.seed; }

// Eight values, the first of which has an index of 8 i8 in its tensor: dropped ones become 0 whatever they were.
__device__ __forceinline__ void drop8(const DropParams& p, uint64_t seed, uint64_t i8, float (&v)[8]) {
  const uint4 q = philox(i8, p.site, seed);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = (w[i] & 0xFFFFu) >= p.threshold ? v[2 * i] * p.factor : 0.f;
    v[2 * i + 1] = (w[i] >> 16) >= p.threshold ? v[2 * i + 1] * p.factor : 0.f;
  }
}

}  // namespace fwn
