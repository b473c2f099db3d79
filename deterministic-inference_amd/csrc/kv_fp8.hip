// The 8-bit KV cache's writer and reader: bf16 K/V rows quantised into the pool, and pool rows
// read back as bf16 (format: kv_fp8.h). Both only move bytes: 16 lanes hold a vector of 128
// (16 bytes of bf16 or 8 of codes a lane), K and V of a token's head side by side in a thread
// so that both loads are in flight, the maximum over the 16 lanes by DPP. Both run at the rate of a
// large copy (4.5 TB/s): 8192 rows are written in 10.2 us, 5.0 TB/s, and 65536 read back in 77 us,
// 5.2; one row takes 1.9 us, the latency of a slot, a row and its maximum.
#include "kv_fp8.h"

namespace sid {
namespace {

constexpr int VEC = 128;               // elements of a head's vector
constexpr int64_t kMaxBlocks = 1 << 22;  // (a grid of 256-thread blocks past 2^32 work-items fails)

// Vector u = (token, head): codes and scales at the token's slot. Slots outside [0, S) are
// skipped, as in reshape_and_cache.
__global__ void __launch_bounds__(256) store_fp8_kernel(
    const bf16_t* __restrict__ k, int64_t ldk, const bf16_t* __restrict__ v, int64_t ldv,
    uint2* __restrict__ k_cache, uint2* __restrict__ v_cache, uint16_t* __restrict__ scales,
    const int64_t* __restrict__ slot_mapping, int64_t vectors, int num_kv_heads,
    int64_t num_slots) {
  const int j = threadIdx.x & 15;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 16;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4); u < vectors;
       u += step) {
    const int64_t t = u / num_kv_heads;
    const int h = static_cast<int>(u % num_kv_heads);
    const int64_t slot = slot_mapping[t];
    if (slot < 0 || slot >= num_slots) continue;  // the vector's 16 lanes together
    const uint4 kk = *reinterpret_cast<const uint4*>(k + t * ldk + h * VEC + 8 * j);
    const uint4 vv = *reinterpret_cast<const uint4*>(v + t * ldv + h * VEC + 8 * j);
    const int64_t vec = slot * num_kv_heads + h;
    float x[8];
    load8(kk, x);
    const int kb = fp8_scale_byte(group_max16(absmax8(x)));
    k_cache[vec * 16 + j] = fp8_encode8(x, kb);
    load8(vv, x);
    const int vb = fp8_scale_byte(group_max16(absmax8(x)));
    v_cache[vec * 16 + j] = fp8_encode8(x, vb);
    if (j == 0) scales[vec] = static_cast<uint16_t>(kb | vb << 8);
  }
}

__device__ __forceinline__ uint4 decode8(uint2 c, uint32_t byte) {
  const float s = fp8_scale(byte);
  const uint2 a = fp8_to_bf16x4(c.x, s), b = fp8_to_bf16x4(c.y, s);
  return make_uint4(a.x, a.y, b.x, b.y);
}

// Vector u = (row i, head) of slot slots[i]; rows of slots outside [0, S) are zeros, as in
// gather_rows.
__global__ void __launch_bounds__(256) gather_fp8_kernel(
    const uint2* __restrict__ k_cache, const uint2* __restrict__ v_cache,
    const uint16_t* __restrict__ scales, const int64_t* __restrict__ slots,
    uint4* __restrict__ k, uint4* __restrict__ v, int64_t vectors, int num_kv_heads,
    int64_t num_slots) {
  const int j = threadIdx.x & 15;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 16;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4); u < vectors;
       u += step) {
    const int64_t slot = slots[u / num_kv_heads];
    uint4 kk = make_uint4(0, 0, 0, 0), vv = kk;
    if (slot >= 0 && slot < num_slots) {
      const int64_t vec = slot * num_kv_heads + u % num_kv_heads;
      const uint2 kc = k_cache[vec * 16 + j];
      const uint2 vc = v_cache[vec * 16 + j];
      const uint32_t s = scales[vec];
      kk = decode8(kc, s & 255u);
      vv = decode8(vc, s >> 8);
    }
    k[u * 16 + j] = kk;
    v[u * 16 + j] = vv;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

unsigned blocks_for(int64_t vectors) {
  const int64_t b = (vectors + 15) / 16;
  return static_cast<unsigned>(b < kMaxBlocks ? b : kMaxBlocks);
}

}  // namespace
}  // namespace sid

using namespace sid;

extern "C" int sid_reshape_and_cache_fp8(const void* k, int64_t ldk, const void* v, int64_t ldv,
                                         void* k_cache, void* v_cache, void* kv_scales,
                                         const int64_t* slot_mapping, int64_t num_tokens,
                                         int num_kv_heads, int head_dim, int64_t num_slots,
                                         void* stream) {
  SID_REQUIRE(num_tokens >= 0, "reshape_and_cache_fp8: negative token count %lld",
              (long long)num_tokens);
  if (num_tokens == 0) return SID_OK;
  SID_REQUIRE(k && v && k_cache && v_cache && kv_scales && slot_mapping,
              "reshape_and_cache_fp8: null pointer");
  SID_REQUIRE(head_dim == VEC, "reshape_and_cache_fp8: head_dim must be %d, got %d", VEC,
              head_dim);
  SID_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 65536, "reshape_and_cache_fp8: bad head count %d",
              num_kv_heads);
  SID_REQUIRE(num_slots > 0, "reshape_and_cache_fp8: empty pool");
  const int64_t row = static_cast<int64_t>(num_kv_heads) * VEC;
  SID_REQUIRE(ldk >= row && ldv >= row && ldk % 8 == 0 && ldv % 8 == 0,
              "reshape_and_cache_fp8: row strides %lld, %lld must be multiples of 8 and at least "
              "%lld", (long long)ldk, (long long)ldv, (long long)row);
  SID_REQUIRE(aligned16(k) && aligned16(v) && aligned16(k_cache) && aligned16(v_cache) &&
                  aligned16(kv_scales),
              "reshape_and_cache_fp8: operands must be 16-byte aligned");
  SID_REQUIRE(num_tokens <= (1ll << 40), "reshape_and_cache_fp8: too many tokens");
  const int64_t vectors = num_tokens * num_kv_heads;
  hipLaunchKernelGGL(store_fp8_kernel, dim3(blocks_for(vectors)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), (const bf16_t*)k, ldk, (const bf16_t*)v,
                     ldv, (uint2*)k_cache, (uint2*)v_cache, (uint16_t*)kv_scales, slot_mapping,
                     vectors, num_kv_heads, num_slots);
  return check_launch("reshape_and_cache_fp8");
}

extern "C" int sid_gather_cache_fp8(const void* k_cache, const void* v_cache,
                                    const void* kv_scales, const int64_t* slots, void* k, void* v,
                                    int64_t n, int num_kv_heads, int head_dim, int64_t num_slots,
                                    void* stream) {
  SID_REQUIRE(n >= 0, "gather_cache_fp8: negative row count %lld", (long long)n);
  if (n == 0) return SID_OK;
  SID_REQUIRE(k_cache && v_cache && kv_scales && slots && k && v, "gather_cache_fp8: null pointer");
  SID_REQUIRE(head_dim == VEC, "gather_cache_fp8: head_dim must be %d, got %d", VEC, head_dim);
  SID_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 65536, "gather_cache_fp8: bad head count %d",
              num_kv_heads);
  SID_REQUIRE(num_slots > 0, "gather_cache_fp8: empty pool");
  SID_REQUIRE(aligned16(k) && aligned16(v) && aligned16(k_cache) && aligned16(v_cache) &&
                  aligned16(kv_scales),
              "gather_cache_fp8: operands must be 16-byte aligned");
  SID_REQUIRE(n <= (1ll << 40), "gather_cache_fp8: too many rows");
  const int64_t vectors = n * num_kv_heads;
  hipLaunchKernelGGL(gather_fp8_kernel, dim3(blocks_for(vectors)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), (const uint2*)k_cache,
                     (const uint2*)v_cache, (const uint16_t*)kv_scales, slots, (uint4*)k,
                     (uint4*)v, vectors, num_kv_heads, num_slots);
  return check_launch("gather_cache_fp8");
}
