// What the C ABI's translation units share (defined in fwn_attn.cu): the thread's last error, the current device's
// multiprocessors, tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "../../include/fwn_attn.h"

namespace fwn {

__attribute__((format(printf, 2, 3))) fwn_status abi_fail(fwn_status s, const char* fmt, ...);
fwn_status abi_ok();
int abi_sms();
// Map over `rank` dimensions (2 or 3) of `dims` elements, the first contiguous, the others `strides` elements apart, with a
// box of 128 bytes (128-byte swizzle) or 64 bytes (64-byte swizzle) by box_rows (by 1).
fwn_status abi_map(CUtensorMap* map, const void* base, int32_t dtype, int rank, const int64_t* dims, const int64_t* strides,
                   int box_bytes, int box_rows);

inline fwn_status abi_cuda_fail(cudaError_t e, const char* what) {
  return abi_fail(FWN_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
}
inline bool abi_float(int32_t t) { return t == FWN_DTYPE_BF16 || t == FWN_DTYPE_F32; }
inline int64_t abi_size(int32_t t) { return t == FWN_DTYPE_F32 ? 4 : t == FWN_DTYPE_BF16 ? 2 : 1; }
inline bool abi_aligned(const void* p, int64_t a) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(a) == 0; }
// Tensors that start off their elements' size would fault in the kernels (NULL, an absent one, passes).
struct AbiTensor {
  const void* p;
  int64_t size;
};
inline fwn_status abi_elements(std::initializer_list<AbiTensor> tensors) {
  for (const AbiTensor& t : tensors)
    if (!abi_aligned(t.p, t.size))
      return abi_fail(FWN_ERR_INVALID_ARGUMENT, "a tensor starts off a multiple of its elements' %lld bytes", static_cast<long long>(t.size));
  return FWN_OK;
}

}  // namespace fwn
