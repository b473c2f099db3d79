// A query row as e4m3 codes, for products with a pool's codes on the matrix units
// (extend_attention_fp8.hip, extend_attention_fp4.hip, decode_attention_fp4.hip).
#pragma once

#include "common.h"
#include "kv_fp8.h"

namespace sid {

typedef int i32x8_v __attribute__((ext_vector_type(8)));

// A query row as two e4m3 vectors: q = 2^e (hi + lo / 16), with q's own e of the pool's rule.
// hi keeps 4 significant bits and lo the other 4 of a bf16 value, so the sum is q exactly for
// elements of 2^-6 2^e and more, and for smaller ones the nearest multiple of 2^-13 2^e. The row's
// largest element m is above 224 2^e: elements from 2^-13.8 m up are exact and the others off by at
// most 2^-21.8 m, which puts a score off by at most 2^-21.8 m sum |k| sm_scale: within what fp32
// sums of m's own products round away unless the keys are zero where q is large. In return two fp8
// products, at the matrix rate of one bf16 product and half its operand reads, take the place of a
// bf16 product with converted codes. A lane holds dims 16 g .. +15 and 64 + 16 g .. +15 of row r.
struct QRow {
  i32x8_v hi, lo;
  int scale;  // E8M0 bytes: hi's in byte 0, lo's in byte 1
};

struct QRaw {
  uint4 u[4];
};
__device__ __forceinline__ QRaw load_q(const bf16_t* qp, int g) {
  QRaw q;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    q.u[i] = *reinterpret_cast<const uint4*>(qp + 64 * (i >> 1) + 16 * g + 8 * (i & 1));
  return q;
}

// Eight elements of a row with the scale byte `byte`; nan: an infinity or a NaN in q, the row's scores
// are NaN.
__device__ __forceinline__ void split_q8(const float (&x)[8], int byte, uint2& hi, uint2& lo) {
  const bool nan = byte == kScaleNaN;
  const float inv = __uint_as_float(static_cast<uint32_t>(nan ? 127 : 254 - byte) << 23);
  hi = fp8_encode8(x, byte);
  float r[8];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint32_t c = w == 0 ? hi.x : hi.y;
    const f32x2_cvt a = __builtin_amdgcn_cvt_pk_f32_fp8(c, false);
    const f32x2_cvt b = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
    r[4 * w] = (x[4 * w] * inv - a.x) * 16.0f;
    r[4 * w + 1] = (x[4 * w + 1] * inv - a.y) * 16.0f;
    r[4 * w + 2] = (x[4 * w + 2] * inv - b.x) * 16.0f;
    r[4 * w + 3] = (x[4 * w + 3] * inv - b.y) * 16.0f;
  }
  lo = nan ? hi : fp8_encode8(r, 127);
}

__device__ __forceinline__ int split_q_scale(int byte) {
  return byte == kScaleNaN ? 127 | 127 << 8 : byte | (byte - 4) << 8;
}

__device__ __forceinline__ QRow split_q(const QRaw& raw, bool row_ok) {
  uint32_t amax = 0;
  float x[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    load8(row_ok ? raw.u[i] : make_uint4(0, 0, 0, 0), x[i]);
    amax = max(amax, absmax8(x[i]));
  }
  {
    const auto p = __builtin_amdgcn_permlane16_swap(amax, amax, false, false);
    amax = max(p[0], p[1]);
    const auto p2 = __builtin_amdgcn_permlane32_swap(amax, amax, false, false);
    amax = max(p2[0], p2[1]);
  }
  const int byte = fp8_scale_byte(amax);
  QRow q;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint2 h, l;
    split_q8(x[i], byte, h, l);
    q.hi[2 * i] = h.x;
    q.hi[2 * i + 1] = h.y;
    q.lo[2 * i] = l.x;
    q.lo[2 * i + 1] = l.y;
  }
  q.scale = split_q_scale(byte);
  return q;
}

// The same for a whole workgroup, once: rows of 128 elements, kQRow bytes apart in the LDS, hi then lo then
// the scales' int. By 16 threads a row, 8 elements each, piece j = their lane % 16; read by lanes (r, g) behind a
// barrier.
constexpr int kQRow = 256 + 16;
__device__ __forceinline__ void split_q_row(const uint4& raw, int j, char* row) {
  float x[8];
  load8(raw, x);
  uint32_t amax = absmax8(x);
  amax = max(amax, __float_as_uint(dpp<DPP_QUAD_XOR1>(__uint_as_float(amax))));
  amax = max(amax, __float_as_uint(dpp<DPP_QUAD_XOR2>(__uint_as_float(amax))));
  amax = max(amax, __float_as_uint(dpp<DPP_HALF_MIRROR>(__uint_as_float(amax))));
  amax = max(amax, __float_as_uint(dpp<DPP_ROW_ROR8>(__uint_as_float(amax))));
  const int byte = fp8_scale_byte(amax);
  uint2 h, l;
  split_q8(x, byte, h, l);
  *reinterpret_cast<uint2*>(row + 8 * j) = h;
  *reinterpret_cast<uint2*>(row + 128 + 8 * j) = l;
  if (j == 0) *reinterpret_cast<int*>(row + 256) = split_q_scale(byte);
}
__device__ __forceinline__ QRow read_q_row(const char* row, int g) {
  QRow q;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x4_v h = *reinterpret_cast<const u32x4_v*>(row + 64 * i + 16 * g);
    const u32x4_v l = *reinterpret_cast<const u32x4_v*>(row + 128 + 64 * i + 16 * g);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      q.hi[4 * i + w] = h[w];
      q.lo[4 * i + w] = l[w];
    }
  }
  q.scale = *reinterpret_cast<const int*>(row + 256);
  return q;
}

}  // namespace sid
