// Dropout's random numbers: Philox4x32-10, the counter-based generator of Salmon, Moraes, Dror and Shaw ("Parallel random
// numbers: as easy as 1, 2, 3", SC 2011). A mask is a function of the value's place in its tensor, so forward and backward
// compute it again instead of keeping it, whatever their tiles, strides or launch shapes.
//
// Value i takes the 16-bit number i % 8 (the words' low halves first) of the counter (i / 8, site, 0) under the 64-bit key
// `seed`, and is dropped where that is below `threshold`. Sixteen bits: one call of the generator, some 80 integer
// instructions, serves the eight values of a thread's access (with 32 bits a value its instructions alone would fill 163,848
// x 512 values' 51 us of memory traffic); the probability is a multiple of 2^-16, and the factor of what is kept is that
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

// The words of the eight values from index 8 i8 of their tensor, and whether value E of them is kept: `least` is the
// threshold in the upper half of a word. All are dropped at a threshold of 65,536, which `least` cannot hold: drop_words
// then gives zeros, below a `least` of all ones.
__device__ __forceinline__ uint32_t drop_least(const DropParams& p) { return p.threshold < 65536u ? p.threshold << 16 : 0xFFFFFFFFu; }
__device__ __forceinline__ uint4 drop_words(const DropParams& p, uint64_t seed, uint64_t i8) {
  return p.threshold < 65536u ? philox(i8, p.site, seed) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ bool drop_keeps(const uint4& q, uint32_t least, int e) {
  const uint32_t w = e < 2 ? q.x : e < 4 ? q.y : e < 6 ? q.z : q.w;
  return (e & 1 ? w : w << 16) >= least;  // the upper half decides: least's lower one is 0 (or both are all ones)
}

}  // namespace fwn
