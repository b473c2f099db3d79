// A K or V vector into a pool of codes, whichever: for the kernels that end in a pool (norm_rope.hip,
// decode_chain.hip).
#pragma once

#include "kv_fp4.h"
#include "kv_fp8.h"

namespace sid {

enum Pool { kPoolBf16, kPoolFp8, kPoolFp4 };

// fp8_store_vector or fp4_store_vector (a vector held by 16 lanes, all active).
template <int POOL>
__device__ __forceinline__ void code_store_vector(float (&x)[8], int j, bool ok, void* codes,
                                                  uint8_t* scales, int64_t vec, int which) {
  static_assert(POOL == kPoolFp8 || POOL == kPoolFp4);
  if constexpr (POOL == kPoolFp8)
    fp8_store_vector(x, j, ok, static_cast<uint2*>(codes), scales, vec, which);
  else
    fp4_store_vector(x, j, ok, static_cast<uint32_t*>(codes), scales, vec, which);
}

}  // namespace sid
