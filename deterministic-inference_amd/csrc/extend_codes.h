// What the extend attention's kernels over pools of codes (extend_attention_fp8.hip: e4m3,
// extend_attention_fp4.hip: e2m1) share beside extend_tile.h: loads into the LDS, a query row as two
// e4m3 vectors, and the order in which workgroups take a ragged batch's query tiles.
#pragma once

#include "extend_tile.h"
#include "kv_fp8.h"

#include <type_traits>

namespace sid {

// Lane l's 16 bytes at its address -> LDS byte lds + 16 l.
__device__ __forceinline__ void dma16(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds)
               : "memory", "m0");
}

typedef int i32x8_v __attribute__((ext_vector_type(8)));

// A V tile in the LDS is bf16, 256 bytes a key, 16-byte piece p of a key at p ^ swv(key): half a wave's
// transpose read takes 32 bytes of 8 keys, which this puts on all banks.
__device__ __forceinline__ int swv(int key) { return 2 * (key & 3) | ((key >> 3) & 1) << 3; }

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

// The other buffer of a pair (an immediate where this one is).
__device__ __forceinline__ int other(int buf) { return 1 - buf; }
template <int B>
__device__ __forceinline__ std::integral_constant<int, 1 - B> other(std::integral_constant<int, B>) {
  return {};
}

// ---- placement ------------------------------------------------------------------------------
//
// The query tiles of a ragged batch walk from one key tile to a whole long context, and a grid ends
// with its last workgroup. So there (`ordered`) the workgroups take the tiles by their keys, most
// first: index i gives the i-th of them, ties by request. That follows from the lengths alone: tile
// m of a request's mt stands at pre + m + 1, pre its prefix in tiles. A wave holds the batch, 64
// requests a step, and finds the i-th place bit by bit. (5 chunks of 90-701 tokens over prefixes of
// 333-5001: 139 -> 125 us; on a uniform batch the search only costs its time in every workgroup,
// 16 x 512 52 -> 57.) Where two workgroups share a CU they are a round of `per_round`
// indices apart, and every other round runs backwards: the longest beside the shortest (125 -> 117).
// Placement only: no result depends on it.
constexpr int kOrderSteps = 4;  // batches up to 256 are ordered

struct Item {
  int b, mtile;  // mtile < 0: there is no such tile
};

// Sum (or, with kMax, maximum) over the wave, in every lane.
template <bool kMax>
__device__ __forceinline__ int wave_reduce(int v) {
  auto op = [](int a, int b) { return kMax ? max(a, b) : a + b; };
  auto step = [](int a, auto ctrl) {
    return __builtin_amdgcn_mov_dpp(a, decltype(ctrl)::value, 0xF, 0xF, false);
  };
  v = op(v, step(v, std::integral_constant<int, DPP_QUAD_XOR1>{}));
  v = op(v, step(v, std::integral_constant<int, DPP_QUAD_XOR2>{}));
  v = op(v, step(v, std::integral_constant<int, DPP_HALF_MIRROR>{}));
  v = op(v, step(v, std::integral_constant<int, DPP_ROW_ROR8>{}));
  return op(op(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
            op(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

template <int ROWS>
__device__ __forceinline__ Item pick_item(int i, bool ordered, int per_round, int batch,
                                          int mtiles, const int32_t* __restrict__ qo_indptr,
                                          const int32_t* __restrict__ kv_indptr) {
  const int round = per_round > 0 ? i / per_round : 0;
  if ((round & 1) != 0 && (round + 1) * per_round <= batch * mtiles)
    i = round * per_round + per_round - 1 - i % per_round;
  if (!ordered) return {i % batch, mtiles - 1 - i / batch};
  const int lane = __lane_id();
  const int steps = ceil_div(batch, 64);
  int pre[kOrderSteps], mt[kOrderSteps], top = 0, total = 0;
#pragma unroll
  for (int s = 0; s < kOrderSteps; ++s) {
    pre[s] = mt[s] = 0;
    if (s >= steps) continue;
    const int b = min(64 * s + lane, batch - 1);
    const int len = qo_indptr[b + 1] - qo_indptr[b];
    const int prefix = kv_indptr[b + 1] - kv_indptr[b] - len;
    pre[s] = max(prefix, 0) / ROWS;
    mt[s] = 64 * s + lane < batch && len > 0 && prefix >= 0 ? ceil_div(len, ROWS) : 0;
    total += mt[s];
    top = max(top, mt[s] > 0 ? pre[s] + mt[s] : 0);
  }
  if (i >= wave_reduce<false>(total)) return {0, -1};
  top = wave_reduce<true>(top);
  auto above = [&](int x) {  // tiles at x or more
    int n = 0;
#pragma unroll
    for (int s = 0; s < kOrderSteps; ++s) {
      if (s >= steps) continue;
      n += max(0, mt[s] - max(0, x - 1 - pre[s]));
    }
    return wave_reduce<false>(n);
  };
  int place = 0;  // the largest x with more than i tiles at x or more
  for (int bit = 31 - __builtin_clz(top | 1); bit >= 0; --bit) {
    const int x = place | 1 << bit;
    if (x <= top && above(x) > i) place = x;
  }
  int left = i - above(place + 1);  // which of the tiles at this place
#pragma unroll
  for (int s = 0; s < kOrderSteps; ++s) {
    if (s >= steps) continue;
    const int m = place - 1 - pre[s];
    uint64_t who = __builtin_amdgcn_ballot_w64(m >= 0 && m < mt[s]);
    const int n = __builtin_popcountll(who);
    if (left >= 0 && left < n) {
      for (; left > 0; --left) who &= who - 1;
      const int at = __builtin_ctzll(who);
      return {64 * s + at, __builtin_amdgcn_readlane(m, at)};
    }
    left -= n;
  }
  return {0, -1};
}

// Workgroups in a grid's first dimension: 2^21 of 512 work-items are a quarter of what it holds, and
// at least one place of 65535 heads.
constexpr int kMaxGridX = 1 << 21;

}  // namespace sid
