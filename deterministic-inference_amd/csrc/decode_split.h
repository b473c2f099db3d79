// What the decode attention's three pool formats (decode_attention.hip: bf16,
// decode_attention_fp8.hip: e4m3 codes, decode_attention_fp4.hip: e2m1 codes) share: the split and segment geometry, the placement
// orders, the merge of a workgroup's waves and the launch of stage 2 (the merge of a request's
// segments, which only sees partials).
#pragma once

#include "common.h"

namespace sid {

constexpr int HEAD_DIM = 128;
constexpr int HKV = 8;              // kv heads (a lane group per head)
constexpr int QPK = 2;              // query heads per kv head
constexpr int HQ = HKV * QPK;
constexpr bool kNonTemporal = true;  // K/V rows are streamed once: +9% HBM throughput
constexpr int kMaxGridSlots = 1024;
constexpr int HEUR_TILE = 32;       // granularity of the heuristic split size
constexpr float NEG_BIG = -1e30f;   // finite "minus infinity" for running maxima
constexpr int kOrderSlotBits = 12;  // wg_order entries: request << 12 | slot
constexpr int kOrderEmpty = 1 << 30;  // wg_order entry flag: the item holds no tokens

__host__ __device__ __forceinline__ int kv_per_split(int seq_len, int n_splits, int fixed_split) {
  if (fixed_split > 0) return fixed_split;
  return ceil_div(ceil_div(seq_len, n_splits), HEUR_TILE) * HEUR_TILE;
}

// The split count of a request when the caller passes no num_splits array: the reference's
// policies restated on the device (sid/kernels/decode_attention.py:65-85): fixed-size splits
// cover the sequence, the heuristic takes one split per 32 tokens up to the grid's split
// count. A request without tokens gets 0 (its output is zeros).
__device__ __forceinline__ int derived_splits(int seq_len, int max_splits, int fixed_split) {
  if (seq_len <= 0) return 0;
  if (fixed_split > 0) return ceil_div(seq_len, fixed_split);
  return min(ceil_div(seq_len, HEUR_TILE), max_splits);
}

// Sum over the 8 lanes of a token group; all 8 lanes get identical bits.
__device__ __forceinline__ float group8_sum(float v) {
  v += dpp<DPP_QUAD_XOR1>(v);
  v += dpp<DPP_QUAD_XOR2>(v);
  v += dpp<DPP_HALF_MIRROR>(v);
  return v;
}

template <bool NT>
__device__ __forceinline__ u32x4_v ld16(const u32x4_v* p) {
  if constexpr (NT) {
    return __builtin_nontemporal_load(p);
  } else {
    return *p;
  }
}

// Token range [start, end) of partial slot y of a request, or false if the slot is empty.
// Slot y is segment j = y % sps of split s = y / sps, with sps = ceil(chunk / seg).
__host__ __device__ __forceinline__ bool segment_range(int seq_len, int n_splits, int fixed_split,
                                                       int seg, int y, int& start, int& end) {
  const int chunk = kv_per_split(seq_len, n_splits, fixed_split);
  const int sl = seg > 0 ? min(seg, chunk) : chunk;
  const int sps = ceil_div(chunk, sl);
  const int s = y / sps;
  if (s >= n_splits) return false;
  const int split_start = s * chunk;
  const int split_end = min(split_start + chunk, seq_len);
  start = split_start + (y % sps) * sl;
  end = min(start + sl, split_end);
  return start < end;
}

// LDS of one stage-1 workgroup: the waves' softmax states, then the merge's scales. The
// accumulators come first and the struct is 16-byte aligned, so their stores and the merge's
// reads are whole 16-byte LDS accesses (with a 4-byte-aligned struct the compiler splits
// them into 4-byte pairs: one request of 1024 tokens took 9.3 -> 10.0 us).
template <int NW>
struct alignas(16) Stage1Lds {
  float acc[NW][HQ][HEAD_DIM];
  float m[NW][HQ];
  float l[NW][HQ];
  float sc[NW][HQ];
  float den[HQ];
  float mx[HQ];
};

// Merge of the waves' states in sh.acc / sh.m / sh.l (complete: a barrier behind their writes)
// into the segment's partial (or, with o_direct, the request's output).
template <int NW>
__device__ __forceinline__ void stage1_merge(Stage1Lds<NW>& sh, int tid, int64_t out_row, int y,
                                             int part_stride, float* __restrict__ part_o,
                                             float* __restrict__ part_lse,
                                             bf16_t* __restrict__ o_direct) {
  auto& s_m = sh.m;
  auto& s_l = sh.l;
  auto& s_acc = sh.acc;
  // Merge the waves in increasing wave order. A wave that saw no token of the segment has
  // m = NEG_BIG and l = 0 and drops out (its scale underflows). One thread per query head
  // takes the max over the waves, every wave's scale and the denominator once; then each
  // thread folds 4 consecutive dims of one head (128-bit LDS reads), with the same
  // per-output operations in the same order as folding every dim on its own.
  auto& s_sc = sh.sc;
  auto& s_den = sh.den;
  auto& s_mx = sh.mx;
  if (tid < HQ) {
    float mx = s_m[0][tid];
#pragma unroll
    for (int w = 1; w < NW; ++w) mx = fmaxf(mx, s_m[w][tid]);
    float den = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float sc = __expf(s_m[w][tid] - mx);
      s_sc[w][tid] = sc;
      den += s_l[w][tid] * sc;
    }
    s_den[tid] = den;
    s_mx[tid] = mx;
  }
  __syncthreads();
  constexpr int Q4 = HEAD_DIM / 4;
  for (int i = tid; i < HQ * Q4; i += NW * 64) {
    const int h = i / Q4;
    const int d0 = (i % Q4) * 4;
    float num[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float sc = s_sc[w][h];
      const float4 a = *reinterpret_cast<const float4*>(&s_acc[w][h][d0]);
      num[0] += a.x * sc;
      num[1] += a.y * sc;
      num[2] += a.z * sc;
      num[3] += a.w * sc;
    }
    const float den = s_den[h];
    const float4 out = make_float4(num[0] / den, num[1] / den, num[2] / den, num[3] / den);
    if (o_direct != nullptr) {
      *reinterpret_cast<uint2*>(&o_direct[(out_row + h) * HEAD_DIM + d0]) =
          make_uint2(pack_bf16x2(out.x, out.y), pack_bf16x2(out.z, out.w));
    } else {
      const int64_t prow = (out_row + h) * part_stride + y;
      *reinterpret_cast<float4*>(&part_o[prow * HEAD_DIM + d0]) = out;
      if (d0 == 0) part_lse[prow] = s_mx[h] + __logf(den);
    }
  }
}

// Stage 2 of a grid of `batch` x grid_slots partial slots, all written by stage 1 (decode_attention.hip).
int launch_decode_stage2(int batch, int grid_slots, const float* part_o, const float* part_lse,
                         int part_stride, void* o, hipStream_t s);

// Argument checks shared by the entry points; `name` begins their messages.
int check_decode_args(const char* name, const void* q, const void* k_cache, const void* v_cache,
                      const int32_t* kv_indptr, const int32_t* kv_indices, void* o, int batch,
                      int num_q_heads, int num_kv_heads, int head_dim, int64_t num_slots,
                      int max_splits, int fixed_split_size);
int check_decode_plan(const char* name, int batch, int segment_size, int grid_slots,
                      const int32_t* wg_order, int workers, const float* part_o,
                      const float* part_lse, int part_batch, int part_stride);

}  // namespace sid
