// The 4-bit KV cache's writer and reader: bf16 K/V rows quantised into the pool, and pool rows
// read back as bf16 (format: kv_fp4.h). Both only move bytes: 16 lanes hold a vector of 128 (16
// bytes of bf16 or 4 of codes a lane; 4 lanes are a block), K and V of a token's head side by side
// in a thread so that both loads are in flight, the maxima over the lanes by DPP. Bound: memory. 8192 rows of
// 8 heads are written in 9.7 us (42 MB, 4.4 TB/s) and read back in as long, 65536 scattered rows read in 69 us
// (340 MB, 4.9 TB/s, four fifths of them written; a large copy reaches 4.6); one row takes 2.
#include "kv_fp4.h"

namespace sid {
namespace {

constexpr int VEC = 128;                 // elements of a head's vector
constexpr int64_t kMaxBlocks = 1 << 22;  // (a grid of 256-thread blocks past 2^32 work-items fails)

// Vector u = (token, head): codes and scales at the token's slot. Slots outside [0, S) are
// skipped, as in reshape_and_cache.
__global__ void __launch_bounds__(256) store_fp4_kernel(
    const bf16_t* __restrict__ k, int64_t ldk, const bf16_t* __restrict__ v, int64_t ldv,
    uint32_t* __restrict__ k_cache, uint32_t* __restrict__ v_cache, uint8_t* __restrict__ scales,
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
    const Fp4Lane ke = fp4_encode_lane(x);
    k_cache[vec * 16 + j] = ke.codes;
    load8(vv, x);
    const Fp4Lane ve = fp4_encode_lane(x);
    v_cache[vec * 16 + j] = ve.codes;
    if ((j & 3) == 0) {
      scales[8 * vec + (j >> 2)] = static_cast<uint8_t>(ke.byte);
      scales[8 * vec + 4 + (j >> 2)] = static_cast<uint8_t>(ve.byte);
    }
  }
}

__device__ __forceinline__ uint4 decode8(uint32_t codes, uint32_t byte) {
  const uint4 x = fp4_to_bf16x8(codes, fp4_scale(byte));
  return byte == kFp4ScaleNaN ? make_uint4(kBf16NaNs, kBf16NaNs, kBf16NaNs, kBf16NaNs) : x;
}

// Vector u = (row i, head) of slot slots[i]; rows of slots outside [0, S) are zeros, as in
// gather_rows.
__global__ void __launch_bounds__(256) gather_fp4_kernel(
    const uint32_t* __restrict__ k_cache, const uint32_t* __restrict__ v_cache,
    const uint2* __restrict__ scales, const int64_t* __restrict__ slots, uint4* __restrict__ k,
    uint4* __restrict__ v, int64_t vectors, int num_kv_heads, int64_t num_slots) {
  const int j = threadIdx.x & 15;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 16;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4); u < vectors;
       u += step) {
    const int64_t slot = slots[u / num_kv_heads];
    uint4 kk = make_uint4(0, 0, 0, 0), vv = kk;
    if (slot >= 0 && slot < num_slots) {
      const int64_t vec = slot * num_kv_heads + u % num_kv_heads;
      const uint32_t kc = k_cache[vec * 16 + j];
      const uint32_t vc = v_cache[vec * 16 + j];
      const uint2 s = scales[vec];
      const int at = 8 * (j >> 2);
      kk = decode8(kc, (s.x >> at) & 255u);
      vv = decode8(vc, (s.y >> at) & 255u);
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

int check_pool(const char* name, const void* k, const void* v, const void* k_cache,
               const void* v_cache, const void* kv_scales, const void* slots, int64_t rows,
               int num_kv_heads, int head_dim, int64_t num_slots) {
  SID_REQUIRE(k && v && k_cache && v_cache && kv_scales && slots, "%s: null pointer", name);
  SID_REQUIRE(head_dim == VEC, "%s: head_dim must be %d, got %d", name, VEC, head_dim);
  SID_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 65536, "%s: bad head count %d", name,
              num_kv_heads);
  SID_REQUIRE(num_slots > 0, "%s: empty pool", name);
  SID_REQUIRE(aligned16(k) && aligned16(v) && aligned16(k_cache) && aligned16(v_cache) &&
                  aligned16(kv_scales),
              "%s: operands must be 16-byte aligned", name);
  SID_REQUIRE(rows <= (1ll << 40), "%s: too many rows", name);
  return SID_OK;
}

}  // namespace
}  // namespace sid

using namespace sid;

extern "C" int sid_reshape_and_cache_fp4(const void* k, int64_t ldk, const void* v, int64_t ldv,
                                         void* k_cache, void* v_cache, void* kv_scales,
                                         const int64_t* slot_mapping, int64_t num_tokens,
                                         int num_kv_heads, int head_dim, int64_t num_slots,
                                         void* stream) {
  const char* name = "reshape_and_cache_fp4";
  SID_REQUIRE(num_tokens >= 0, "%s: negative token count %lld", name, (long long)num_tokens);
  if (num_tokens == 0) return SID_OK;
  const int rc = check_pool(name, k, v, k_cache, v_cache, kv_scales, slot_mapping, num_tokens,
                            num_kv_heads, head_dim, num_slots);
  if (rc != SID_OK) return rc;
  const int64_t row = static_cast<int64_t>(num_kv_heads) * VEC;
  SID_REQUIRE(ldk >= row && ldv >= row && ldk % 8 == 0 && ldv % 8 == 0,
              "%s: row strides %lld, %lld must be multiples of 8 and at least %lld", name,
              (long long)ldk, (long long)ldv, (long long)row);
  const int64_t vectors = num_tokens * num_kv_heads;
  hipLaunchKernelGGL(store_fp4_kernel, dim3(blocks_for(vectors)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), (const bf16_t*)k, ldk, (const bf16_t*)v,
                     ldv, (uint32_t*)k_cache, (uint32_t*)v_cache, (uint8_t*)kv_scales,
                     slot_mapping, vectors, num_kv_heads, num_slots);
  return check_launch(name);
}

extern "C" int sid_gather_cache_fp4(const void* k_cache, const void* v_cache,
                                    const void* kv_scales, const int64_t* slots, void* k, void* v,
                                    int64_t n, int num_kv_heads, int head_dim, int64_t num_slots,
                                    void* stream) {
  const char* name = "gather_cache_fp4";
  SID_REQUIRE(n >= 0, "%s: negative row count %lld", name, (long long)n);
  if (n == 0) return SID_OK;
  const int rc = check_pool(name, k, v, k_cache, v_cache, kv_scales, slots, n, num_kv_heads,
                            head_dim, num_slots);
  if (rc != SID_OK) return rc;
  const int64_t vectors = n * num_kv_heads;
  hipLaunchKernelGGL(gather_fp4_kernel, dim3(blocks_for(vectors)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), (const uint32_t*)k_cache,
                     (const uint32_t*)v_cache, (const uint2*)kv_scales, slots, (uint4*)k,
                     (uint4*)v, vectors, num_kv_heads, num_slots);
  return check_launch(name);
}
