// The 8-bit KV cache's number format, shared by the kernels that write it, read it back and
// attend over it (kv_fp8.hip, norm_rope.hip, decode_chain.hip, decode_attention_fp8.hip,
// extend_attention_fp8.hip).
//
// A K (or V) vector of one token's head (128 elements) is 128 e4m3 codes c and one power of
// two 2^e, stored as the E8M0 byte e + 127: x ~ c 2^e with the smallest e for which
// max |x| <= 448 2^e (448 is e4m3's largest value). A power of two costs a floating-point code
// no accuracy but at the bottom of its range (below 2^-14.8 of the vector's maximum), and it
// makes x 2^-e exact, so a stored value is rounded once; c 2^e is a bf16 value exactly, so
// reading back rounds nothing. e is clamped to [-117, 119]: there every c 2^e is zero or a
// normal finite bf16 value (codes saturate at 448 above, vanish below). e4m3 has no infinity:
// a vector that holds an infinity or a NaN is stored as NaN as a whole, with NaN codes and the
// byte 255 (E8M0's NaN), so that a reader which must not let a hidden key's NaN through (0 NaN is
// NaN) sees it in the byte.
//
// The pool: k_cache, v_cache [S, HKV, 128] codes, kv_scales [S, HKV, 2] bytes (K's, V's): both
// scales of a head are one 2-byte load.
#pragma once

#include "rowmath.h"

namespace sid {

constexpr int kScaleMin = 127 - 117, kScaleMax = 127 + 119, kScaleNaN = 255;
constexpr uint32_t kCodesNaN = 0x7f7f7f7fu;
constexpr float kCodeMax = 448.0f;

typedef __bf16 bf16x2_cvt __attribute__((ext_vector_type(2)));
typedef float f32x2_cvt __attribute__((ext_vector_type(2)));

// The scale byte of a vector whose largest magnitude has the fp32 bits `amax` (sign cleared;
// compared as integers, so infinity and NaN are the largest): 448 = 1.75 2^8, so the exponent
// field less 8, one more where the mantissa is above 1.75.
__device__ __forceinline__ int fp8_scale_byte(uint32_t amax) {
  const int b = static_cast<int>((amax + 0x1fffffu) >> 23) - 8;
  return amax >= 0x7f800000u ? kScaleNaN : min(max(b, kScaleMin), kScaleMax);
}

// 2^e of a scale byte.
__device__ __forceinline__ float fp8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight values of a vector with scale byte `byte` to eight codes (round to nearest even).
__device__ __forceinline__ uint2 fp8_encode8(const float (&x)[8], int byte) {
  if (byte == kScaleNaN) return make_uint2(kCodesNaN, kCodesNaN);
  const float inv = __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i] * inv, -kCodeMax, kCodeMax);
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
  return make_uint2(static_cast<uint32_t>(lo), static_cast<uint32_t>(hi));
}

__device__ __forceinline__ uint32_t absmax8(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return m;
}

// Integer maximum over an aligned group of 16 lanes (every lane active; all get it).
__device__ __forceinline__ uint32_t group_max16(uint32_t v) {
  auto step = [](uint32_t a, float b) { return max(a, __float_as_uint(b)); };
  v = step(v, dpp<DPP_QUAD_XOR1>(__uint_as_float(v)));
  v = step(v, dpp<DPP_QUAD_XOR2>(__uint_as_float(v)));
  v = step(v, dpp<DPP_HALF_MIRROR>(__uint_as_float(v)));
  v = step(v, dpp<DPP_ROW_ROR8>(__uint_as_float(v)));
  return v;
}

// Four codes (one 32-bit word) times 2^e as four packed bf16 values: exact.
__device__ __forceinline__ uint2 fp8_to_bf16x4(uint32_t w, float scale) {
  const bf16x2_cvt lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false);
  const bf16x2_cvt hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true);
  return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// A vector held by 16 lanes (8 values each, all active; j: the lane's place) into the pool:
// codes, and the scale of K (which = 0) or V (1). Values are rounded to bf16 first, so a fused
// producer stores what it would have handed to reshape_and_cache_fp8. `ok`: the slot exists.
__device__ __forceinline__ void fp8_store_vector(float (&x)[8], int j, bool ok, uint2* codes,
                                                 uint8_t* scales, int64_t vec, int which) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = round_bf16(x[i]);
  const int byte = fp8_scale_byte(group_max16(absmax8(x)));
  if (!ok) return;
  codes[vec * 16 + j] = fp8_encode8(x, byte);
  if (j == 0) scales[2 * vec + which] = static_cast<uint8_t>(byte);
}

}  // namespace sid
