// What the extend attention's kernels for the three pool formats (extend_attention.hip: bf16,
// extend_attention_fp8.hip: e4m3 codes, extend_attention_fp4.hip: e2m1 codes) share: the tile sizes, a
// row's folded softmax state, its fold and its output, the lane reductions, the host's plan and the merge
// of a fan-out. The tile arithmetic is each kernel's own, and so are their bits: the kernels over codes
// take S on the codes with q as e4m3, sum l by lanes and fold every 512 keys instead of 256.
#pragma once

#include "common.h"

namespace sid {

constexpr int D = 128;
constexpr int BN = 64;          // keys per tile
constexpr int BQ = 32;          // query positions per workgroup (x 2 heads = 64 rows)
constexpr float NEG_BIG = -1e30f;
constexpr float LOG2E = 1.4426950408889634f;
// Slack of the lazy softmax maximum, in log2 units: scores up to LAZY_T above the row's
// reference maximum are taken without moving it (the 4-bit pool's kernel has a slack of its own).
constexpr float LAZY_T = 8.0f;

// 2^x by the hardware instruction (v_exp_f32): results that would be denormal may flush to zero. The
// argument is at most LAZY_T over bf16 and 8-bit pools. The 4-bit pool's kernel bounds it only after
// the fact, by the sum that it grows: there it may be any number, and one that is too large must give a
// large result or infinity.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Reductions over lanes l and l ^ 16 (l ^ 32): v_permlane16/32_swap hand each lane the
// values of both lanes of its pair as (lower lane's, upper lane's), so both lanes compute
// the same expression on the same operands (identical bits) without an LDS round trip.
__device__ __forceinline__ float pair16_max(float v) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float pair32_max(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float pair16_sum(float v) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
__device__ __forceinline__ float pair32_sum(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

typedef short s16x4_v __attribute__((ext_vector_type(4)));
typedef short s16x8_v __attribute__((ext_vector_type(8)));

typedef __attribute__((address_space(3))) char* lds_char_t;

// acc / l (l > 0), shared by every path that divides: y = 1 / l rounded, q = acc y, then one
// correction (Markstein: the quotient correctly rounded), 5 operations for each of a row's
// dims instead of a division's 12. An infinite or NaN q stays.
__device__ __forceinline__ float div_row(float acc, float l, float y) {
  const float q = acc * y;
  const float c = __builtin_fmaf(__builtin_fmaf(-q, l, acc), y, q);
  return __builtin_fabsf(q) < INFINITY ? c : q;
}

// Per-lane softmax state of one query row (the lane's 32 output dims).
struct RowState {
  float m;
  float l;
  f32x4_v acc[8];
};

// The fold of a split's state into a row's: its per-row scalars and its elementwise step, shared by
// every path that folds.
struct FoldScale {
  float mn, alpha, beta;
};
__device__ __forceinline__ FoldScale fold_scale(float run_m, float m) {
  const float mn = fmaxf(run_m, m);
  return {mn, exp2_fast(run_m - mn), exp2_fast(m - mn)};
}
// Written as one explicit fma over a separately rounded product, so the compiler has no
// contraction choice to make differently in different kernels.
__device__ __forceinline__ float fold_elem(float run, float part, const FoldScale& f) {
  return __builtin_fmaf(run, f.alpha, part * f.beta);
}

// The row's output: acc / l rounded to bf16 (this lane: dims 16 db + 4 g .. +3).
__device__ __forceinline__ void store_row(bf16_t* op, const RowState& run, int g) {
  const float y = 1.0f / run.l;
#pragma unroll
  for (int db = 0; db < 8; ++db) {
    const f32x4_v a = run.acc[db];
    uint2 u;
    u.x = pack_bf16x2(div_row(a[0], run.l, y), div_row(a[1], run.l, y));
    u.y = pack_bf16x2(div_row(a[2], run.l, y), div_row(a[3], run.l, y));
    *reinterpret_cast<uint2*>(op + 16 * db + 4 * g) = u;
  }
}

constexpr int kTileBytes = BN * D * 2;  // one K or V tile

// What a fan-out kernel leaves to the merge for each (row, head): how many splits have its state.
// Rows of a request that is left out get 0, and the merge leaves them as they are, as a kernel that
// walks the keys does. By the threads of the workgroup that has the split 0 of the rows' tile.
__device__ __forceinline__ void skip_rows(int32_t* part_n, int q_start, int from, int to,
                                          int num_q_heads, int h_kv) {
  for (int i = threadIdx.x; i < 2 * (to - from); i += blockDim.x)
    part_n[static_cast<int64_t>(q_start + from + (i >> 1)) * num_q_heads + 2 * h_kv + (i & 1)] = 0;
}

// ---- host side (extend_attention.hip) -----------------------------------------------------

// Query positions (32 or 64) of a workgroup that walks all keys of its rows.
int extend_prefill_rows(int batch, int64_t total_q, int num_kv_heads, int max_extend_len);

// The launch of a call, worked out once for all formats: what is checked, whether the splits fan
// out over workgroups (the caller's rule asks for `need` bytes and the workspace has them), the
// grid.
struct ExtendPlan {
  int rc;             // SID_OK or the error
  bool empty;         // nothing to do
  bool fanout;
  int rows;           // 32 or 64 query positions a workgroup (fan-out: 32)
  int mtiles, splits;
  unsigned grid_x;    // workgroups over the requests (padded for ragged batches)
  int64_t items;      // (query row, head) pairs
  float* part_a;
  float* part_ml;
  int32_t* part_n;
};
ExtendPlan extend_plan(const char* name, const void* q, const void* k_cache, const void* v_cache,
                       const int32_t* qo_indptr, const int32_t* kv_indptr,
                       const int32_t* kv_indices, const void* o, int batch, int64_t total_q,
                       int num_q_heads, int num_kv_heads, int head_dim, int64_t num_slots,
                       int max_extend_len, int max_kv_len, int split_keys, int64_t need,
                       void* workspace, int64_t workspace_bytes);

// The fan-out's second launch: the saved split states of every item of the sequences' rows folded
// in order.
int extend_merge(const char* name, const ExtendPlan& p, const int32_t* qo_indptr, int batch,
                 int num_q_heads, void* o, hipStream_t s);

}  // namespace sid
