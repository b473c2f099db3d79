// A K or V vector into a pool of codes, whichever: for the kernels that end in a pool (norm_rope.hip,
// decode_chain.hip). Over a 4-bit pool qkv_post of 8192 rows takes 28 us (110 MB; bf16 34 us for 135) and of
// 64 rows of partials 3.4; rmsnorm_qkv_post of 64 rows 8.7 (8.4 MB of weights; latency), both as over bf16.
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
