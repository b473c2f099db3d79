// The 4-bit KV cache's number format, shared by the kernels that write it, read it back and
// attend over it (kv_fp4.hip, norm_rope.hip, decode_chain.hip, decode_attention_fp4.hip,
// extend_attention_fp4.hip).
//
// A K (or V) vector of one token's head (128 elements) is four blocks of 32 consecutive elements. A
// block is 32 e2m1 codes c (+-0, 0.5, 1, 1.5, 2, 3, 4, 6; two a byte, the even element in the low
// half) and one power of two 2^e, stored as the E8M0 byte e + 127: x ~ c 2^e with the smallest e
// for which max |x| <= 6 2^e. That is the block that gfx950's matrix products take as it lies in
// memory: a lane's 32 codes are 16 bytes with one scale of their own. x 2^-e is exact, so a stored
// value is rounded once, by at most 2^e / 4 where |x| < 2^(e+1), 2^e / 2 up to 2^(e+2), 2^e above;
// c 2^e is a bf16 value exactly, so reading back rounds nothing. e is clamped to [-125, 125]: there
// every c 2^e is zero or a normal finite bf16 value (codes saturate at 6 above, vanish below).
// Neither e2m1 nor a block has a place for infinity: a vector that holds an infinity or a NaN is
// stored as NaN as a whole, with the byte 255 (E8M0's NaN) in all its blocks.
//
// The pool: k_cache, v_cache [S, HKV, 64] bytes of codes, kv_scales [S, HKV, 2, 4] bytes (K's four
// blocks, V's four): all scales of a head are one 8-byte load.
#pragma once

#include "rowmath.h"

namespace sid {

constexpr int kFp4Block = 32;
constexpr int kFp4ScaleMin = 127 - 125, kFp4ScaleMax = 127 + 125, kFp4ScaleNaN = 255;
constexpr uint32_t kFp4CodesNaN = 0x77777777u;  // (what the byte says; the codes are not read)
constexpr uint32_t kBf16NaNs = 0x7fc07fc0u;

typedef __bf16 bf16x2_fp4 __attribute__((ext_vector_type(2)));
typedef float f32x2_fp4 __attribute__((ext_vector_type(2)));

// The scale byte of a block whose largest magnitude has the fp32 bits `amax` (sign cleared) and is
// finite: 6 = 1.5 2^2, so the exponent field less 2, one more where the mantissa is above 1.5.
__device__ __forceinline__ int fp4_scale_byte(uint32_t amax) {
  const int b = static_cast<int>((amax + 0x3fffffu) >> 23) - 2;
  return min(max(b, kFp4ScaleMin), kFp4ScaleMax);
}

// 2^e of a scale byte (of 255: an infinity's bits, which the conversions below make NaN).
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight values of a block to eight codes: x 2^-e, to nearest even, saturating, by the conversion
// instruction (its scale operand gives the power of two by its exponent).
__device__ __forceinline__ uint32_t fp4_encode8(const float (&x)[8], int byte) {
  const float s = fp4_scale(byte);
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], s, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], s, 3);
}

__device__ __forceinline__ uint32_t fp4_absmax8(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return m;
}

// Eight codes (one 32-bit word) times 2^e as eight packed bf16 values: exact.
__device__ __forceinline__ uint4 fp4_to_bf16x8(uint32_t w, float scale) {
  return make_uint4(
      __builtin_bit_cast(uint32_t, (bf16x2_fp4)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
      __builtin_bit_cast(uint32_t, (bf16x2_fp4)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
      __builtin_bit_cast(uint32_t, (bf16x2_fp4)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
      __builtin_bit_cast(uint32_t, (bf16x2_fp4)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3)));
}

// The codes and the scale byte of a lane's eight values, in a vector held by an aligned group of 16
// lanes, four to a block (every lane active).
struct Fp4Lane {
  uint32_t codes;
  int byte;
};
__device__ __forceinline__ Fp4Lane fp4_encode_lane(const float (&x)[8]) {
  auto step = [](uint32_t a, float b) { return max(a, __float_as_uint(b)); };
  uint32_t m = fp4_absmax8(x);
  m = step(m, dpp<DPP_QUAD_XOR1>(__uint_as_float(m)));
  m = step(m, dpp<DPP_QUAD_XOR2>(__uint_as_float(m)));  // the block's
  uint32_t all = step(m, dpp<DPP_HALF_MIRROR>(__uint_as_float(m)));
  all = step(all, dpp<DPP_ROW_ROR8>(__uint_as_float(all)));  // the vector's
  const int byte = fp4_scale_byte(m);
  const bool nan = all >= 0x7f800000u;  // compared as integers: infinity and NaN are the largest
  return {nan ? kFp4CodesNaN : fp4_encode8(x, byte), nan ? kFp4ScaleNaN : byte};
}

// A vector held by 16 lanes (8 values each, all active; j: the lane's place) into the pool: codes,
// and the scales of K (which = 0) or V (1). Values are rounded to bf16 first, so a fused producer
// stores what it would have handed to reshape_and_cache_fp4. `ok`: the slot exists.
__device__ __forceinline__ void fp4_store_vector(float (&x)[8], int j, bool ok, uint32_t* codes,
                                                 uint8_t* scales, int64_t vec, int which) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = round_bf16(x[i]);
  const Fp4Lane e = fp4_encode_lane(x);
  if (!ok) return;
  codes[vec * 16 + j] = e.codes;
  if ((j & 3) == 0) scales[8 * vec + 4 * which + (j >> 2)] = static_cast<uint8_t>(e.byte);
}

}  // namespace sid
