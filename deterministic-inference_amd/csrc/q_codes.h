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
  const bool nan = byte == kScaleNaN;  // an infinity or a NaN in q: the row's scores are NaN
  const float inv = __uint_as_float(static_cast<uint32_t>(nan ? 127 : 254 - byte) << 23);
  QRow q;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint2 h = fp8_encode8(x[i], byte);
    float r[8];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const uint32_t c = w == 0 ? h.x : h.y;
      const f32x2_cvt a = __builtin_amdgcn_cvt_pk_f32_fp8(c, false);
      const f32x2_cvt b = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
      r[4 * w] = (x[i][4 * w] * inv - a.x) * 16.0f;
      r[4 * w + 1] = (x[i][4 * w + 1] * inv - a.y) * 16.0f;
      r[4 * w + 2] = (x[i][4 * w + 2] * inv - b.x) * 16.0f;
      r[4 * w + 3] = (x[i][4 * w + 3] * inv - b.y) * 16.0f;
    }
    const uint2 l = nan ? h : fp8_encode8(r, 127);
    q.hi[2 * i] = h.x;
    q.hi[2 * i + 1] = h.y;
    q.lo[2 * i] = l.x;
    q.lo[2 * i + 1] = l.y;
  }
  q.scale = nan ? 127 | 127 << 8 : byte | (byte - 4) << 8;
  return q;
}

}  // namespace sid
