// What the extend attention's kernels over pools of codes (extend_attention_fp8.hip: e4m3,
// extend_attention_fp4.hip: e2m1) share beside extend_tile.h and q_codes.h: loads into the LDS and the order in which workgroups
// take a ragged batch's query tiles.
#pragma once

#include "extend_tile.h"
#include "q_codes.h"

#include <type_traits>

namespace sid {

// Lane l's 16 bytes at its address -> LDS byte lds + 16 l.
__device__ __forceinline__ void dma16(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds)
               : "memory", "m0");
}

// A V tile in the LDS is bf16, 256 bytes a key, 16-byte piece p of a key at p ^ swv(key): half a wave's
// transpose read takes 32 bytes of 8 keys, which this puts on all banks.
__device__ __forceinline__ int swv(int key) { return 2 * (key & 3) | ((key >> 3) & 1) << 3; }

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
