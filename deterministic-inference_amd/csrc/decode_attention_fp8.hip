// Split-KV paged decode attention over the 8-bit pool (format: kv_fp8.h), gfx950.
//
// The partition into splits and segments, the placement orders, the waves' merge and stage 2
// are decode_attention.hip's (decode_split.h); only what a wave does with a token's row differs:
//   * a row of K (V) is 8 heads x 128 codes = 1 KiB, one 16-byte load of a wave: lane group g
//     (8 lanes) owns kv head g and its two query heads, lane `sub` dims 16 sub .. 16 sub + 15;
//     the two scales of (token, head) come as one 2-byte load, 16 bytes a token;
//   * codes are converted without their scale (exact), the powers of two enter where a token
//     has one value a head: s = (q . c_k) (2^e_k sm_scale) and o += (p 2^e_v) c_v.
//
// Bound: the pool's rows, 2064 bytes a token. A wave asks for 4 tokens' rows (8 KiB), then
// computes on the 4 before: its conversions and dot products take about half as long as the rows
// take to come, and with loads and math in turn neither hides the other (128 requests of 4096
// keys 173.2 -> 169.3 us with the rows a step ahead, 64 of 2048 48.9 -> 47.0, 32 ragged ones of
// 128-4096 31.6 -> 29.2). 4 tokens an iteration: with 8 the wave holds 209 registers and one
// workgroup fits a CU, with 2 too little is in flight (128 x 4096: 172 us with two workgroups a
// CU, 203 with a plan of one). 128 x 4096 keys: 166 us, 6.5 TB/s, with the
// merge, where a plain read of the same size reaches 6.0-6.5; 1 x 1024: 9.9 us in a graph, the chain
// of launch, slots, rows, merge and stage 2's launch (the bf16 pool's kernel 10.3 in the same run).
#include "decode_split.h"
#include "kv_fp8.h"

namespace sid {
namespace {

__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_v, a),
                                         __builtin_bit_cast(bf16x2_v, b), c, false);
}

constexpr int TPL = 4;  // tokens per wave iteration

struct TileRegs {
  u32x4_v k[TPL];
  u32x4_v v[TPL];
  uint16_t sc[TPL];
};

// The partial attention of request b over partial slot y (a segment of one split), by one
// workgroup of NW waves taking TPL tokens per wave iteration. Every exit is
// workgroup-uniform.
template <int NW>
__device__ __forceinline__ void stage1_item(
    Stage1Lds<NW>& sh, int b, int y, const bf16_t* __restrict__ q,
    const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
    const uint16_t* __restrict__ kv_scales, const int32_t* __restrict__ kv_indptr,
    const int32_t* __restrict__ kv_indices, const int32_t* __restrict__ num_splits,
    int max_splits, int fixed_split, int seg, float sm_scale, int64_t num_slots, int part_stride,
    float* __restrict__ part_o, float* __restrict__ part_lse, bf16_t* __restrict__ o_direct) {
  constexpr int IT = NW * TPL;  // tokens per workgroup iteration
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int grp = lane >> 3;  // kv head
  const int sub = lane & 7;

  const int kv_base = kv_indptr[b];
  const int seq_len = kv_indptr[b + 1] - kv_base;
  const int n_splits = num_splits != nullptr ? num_splits[b]
                                             : derived_splits(seq_len, max_splits, fixed_split);
  const int64_t out_row = static_cast<int64_t>(b) * HQ;
  int start = 0, end = 0;
  if (n_splits <= 0 || seq_len <= 0 ||
      !segment_range(seq_len, n_splits, fixed_split, seg, y, start, end)) {
    // A slot with no tokens: zeros where there is no stage 2 to write them, else the mark that
    // stage 2 looks for.
    if (o_direct != nullptr) {
      if (y == 0) {
        for (int i = tid; i < HQ * HEAD_DIM; i += NW * 64) o_direct[out_row * HEAD_DIM + i] = 0;
      }
    } else if (tid < HQ) {
      part_lse[(out_row + tid) * part_stride + y] = NEG_BIG;
    }
    return;
  }

  // Query heads 2 grp and 2 grp + 1: the lane's 16 dims, packed bf16.
  u32x4_v qv[QPK][2];
#pragma unroll
  for (int h = 0; h < QPK; ++h) {
    const u32x4_v* qb =
        reinterpret_cast<const u32x4_v*>(q + (out_row + QPK * grp + h) * HEAD_DIM + 16 * sub);
    qv[h][0] = qb[0];
    qv[h][1] = qb[1];
  }
  float m[QPK], l[QPK], acc[QPK][16];
#pragma unroll
  for (int h = 0; h < QPK; ++h) {
    m[h] = NEG_BIG;
    l[h] = 0.0f;
#pragma unroll
    for (int d = 0; d < 16; ++d) acc[h][d] = 0.0f;
  }

  const int32_t* idx = kv_indices + kv_base;
  auto load_idx = [&](int t0, int32_t (&raw)[TPL]) {
#pragma unroll
    for (int t = 0; t < TPL; ++t) raw[t] = idx[min(t0 + t, end - 1)];
  };
  // Positions past the segment's end load its last token again and get weight 0.
  auto load_tile = [&](int t0, const int32_t (&raw)[TPL], bool (&ok)[TPL], TileRegs& r) {
#pragma unroll
    for (int t = 0; t < TPL; ++t) {
      int64_t sv = static_cast<int64_t>(raw[t]);
      if (sv < 0 || sv >= num_slots) sv = 0;
      ok[t] = t0 + t < end;
      r.k[t] = ld16<true>(reinterpret_cast<const u32x4_v*>(k_cache + sv * (HKV * HEAD_DIM)) + lane);
      r.v[t] = ld16<true>(reinterpret_cast<const u32x4_v*>(v_cache + sv * (HKV * HEAD_DIM)) + lane);
      r.sc[t] = kv_scales[sv * HKV + grp];
    }
    __builtin_amdgcn_sched_barrier(0);  // (as in decode_attention.hip: all loads go out first)
  };
  auto compute = [&](const bool (&ok)[TPL], const TileRegs& r) {
    float sc[QPK][TPL];
#pragma unroll
    for (int t = 0; t < TPL; ++t) {
      float s[QPK] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint2 kc = fp8_to_bf16x4(r.k[t][i], 1.0f);
#pragma unroll
        for (int h = 0; h < QPK; ++h) {
          s[h] = dot2(qv[h][i >> 1][2 * (i & 1)], kc.x, s[h]);
          s[h] = dot2(qv[h][i >> 1][2 * (i & 1) + 1], kc.y, s[h]);
        }
      }
      const float ks = fp8_scale(r.sc[t] & 255u) * sm_scale;
#pragma unroll
      for (int h = 0; h < QPK; ++h) sc[h][t] = group8_sum(s[h]) * ks;
    }
#pragma unroll
    for (int h = 0; h < QPK; ++h) {
      float tmax = NEG_BIG;
#pragma unroll
      for (int t = 0; t < TPL; ++t)
        if (ok[t]) tmax = fmaxf(tmax, sc[h][t]);
      const float mn = fmaxf(m[h], tmax);
      const float rs = __expf(m[h] - mn);
      float psum = 0.0f;
#pragma unroll
      for (int t = 0; t < TPL; ++t) {
        sc[h][t] = ok[t] ? __expf(sc[h][t] - mn) : 0.0f;
        psum += sc[h][t];
      }
      l[h] = l[h] * rs + psum;
      m[h] = mn;
      if (__builtin_amdgcn_ballot_w64(rs != 1.0f) != 0) {
#pragma unroll
        for (int d = 0; d < 16; ++d) acc[h][d] *= rs;
      }
    }
#pragma unroll
    for (int t = 0; t < TPL; ++t) {
      const float vs = fp8_scale(r.sc[t] >> 8);
      float w[QPK];
#pragma unroll
      for (int h = 0; h < QPK; ++h) w[h] = sc[h][t] * vs;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2_cvt a = __builtin_amdgcn_cvt_pk_f32_fp8(r.v[t][i], false);
        const f32x2_cvt c = __builtin_amdgcn_cvt_pk_f32_fp8(r.v[t][i], true);
#pragma unroll
        for (int h = 0; h < QPK; ++h) {
          acc[h][4 * i + 0] += w[h] * a.x;
          acc[h][4 * i + 1] += w[h] * a.y;
          acc[h][4 * i + 2] += w[h] * c.x;
          acc[h][4 * i + 3] += w[h] * c.y;
        }
      }
    }
  };

  // Rows are loaded one iteration ahead of their math, their slots two.
  int32_t raw[TPL];
  TileRegs r;
  bool ok[TPL];
  int t0 = start + wave * TPL;
  load_idx(t0, raw);
  load_tile(t0, raw, ok, r);
  load_idx(t0 + IT, raw);
  for (; t0 + IT < end; t0 += IT) {
    TileRegs next;
    bool next_ok[TPL];
    load_tile(t0 + IT, raw, next_ok, next);
    load_idx(t0 + 2 * IT, raw);
    compute(ok, r);
    r = next;
#pragma unroll
    for (int t = 0; t < TPL; ++t) ok[t] = next_ok[t];
  }
  if (t0 < end) compute(ok, r);

#pragma unroll
  for (int h = 0; h < QPK; ++h) {
    const int hq = QPK * grp + h;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<float4*>(&sh.acc[wave][hq][16 * sub + 4 * j]) =
          make_float4(acc[h][4 * j], acc[h][4 * j + 1], acc[h][4 * j + 2], acc[h][4 * j + 3]);
    if (sub == 0) {
      sh.m[wave][hq] = m[h];
      sh.l[wave][hq] = l[h];
    }
  }
  __syncthreads();
  stage1_merge<NW>(sh, tid, out_row, y, part_stride, part_o, part_lse, o_direct);
}

// Grid form and worker form, as in decode_attention.hip: workgroup (b, y), or the entry of
// wg_order at its linear id; or the items that wg_order deals to each of `gridDim.x` workers
// (order entries i, i + workers, ...; from the first one flagged empty on, all are).
template <int NW, bool WORKER>
__global__ void __launch_bounds__(NW * 64) decode_fp8_stage1_kernel(
    const bf16_t* __restrict__ q, const uint8_t* __restrict__ k_cache,
    const uint8_t* __restrict__ v_cache, const uint16_t* __restrict__ kv_scales,
    const int32_t* __restrict__ kv_indptr, const int32_t* __restrict__ kv_indices,
    const int32_t* __restrict__ num_splits, int max_splits, int fixed_split, int seg,
    float sm_scale, int64_t num_slots, int part_stride, float* __restrict__ part_o,
    float* __restrict__ part_lse, bf16_t* __restrict__ o_direct,
    const int32_t* __restrict__ wg_order, int batch, int grid_slots) {
  __shared__ Stage1Lds<NW> sh;
  auto item = [&](int b, int y) {
    stage1_item<NW>(sh, b, y, q, k_cache, v_cache, kv_scales, kv_indptr, kv_indices,
                         num_splits, max_splits, fixed_split, seg, sm_scale, num_slots,
                         part_stride, part_o, part_lse, o_direct);
  };
  constexpr int kSlotMask = (1 << kOrderSlotBits) - 1;
  if constexpr (!WORKER) {
    int b = blockIdx.x;
    int y = blockIdx.y;
    if (wg_order != nullptr) {
      const int packed = wg_order[blockIdx.x + blockIdx.y * gridDim.x] & ~kOrderEmpty;
      b = static_cast<int>(static_cast<uint32_t>(packed) >> kOrderSlotBits);
      y = packed & kSlotMask;
      if (b >= batch || y >= grid_slots) return;
    }
    item(b, y);
  } else {
    const int n_items = batch * grid_slots;
    const int W = static_cast<int>(gridDim.x);
    int i = static_cast<int>(blockIdx.x);
    for (; i < n_items; i += W) {
      const int packed = wg_order[i];  // workgroup-uniform
      if (packed & kOrderEmpty) break;
      const int b = static_cast<int>(static_cast<uint32_t>(packed) >> kOrderSlotBits);
      const int y = packed & kSlotMask;
      if (b < batch && y < grid_slots) item(b, y);
      __syncthreads();  // the item's merge reads of the LDS are done before the next one's writes
    }
    const int rest = i < n_items ? (n_items - i + W - 1) / W : 0;
    for (int t = threadIdx.x; t < rest * HQ; t += NW * 64) {
      const int packed = wg_order[i + (t / HQ) * W] & ~kOrderEmpty;
      const int b = static_cast<int>(static_cast<uint32_t>(packed) >> kOrderSlotBits);
      const int y = packed & kSlotMask;
      if (b < batch && y < grid_slots)
        part_lse[(static_cast<int64_t>(b) * HQ + t % HQ) * part_stride + y] = NEG_BIG;
    }
  }
}

constexpr int kNumVariants = 4;

}  // namespace
}  // namespace sid

using namespace sid;

extern "C" int sid_flash_decode_fp8_fwd(
    const void* q, const void* k_cache, const void* v_cache, const void* kv_scales,
    const int32_t* kv_indptr, const int32_t* kv_indices, const int32_t* num_splits, int batch,
    int num_q_heads, int num_kv_heads, int head_dim, int64_t num_slots, int max_splits,
    int fixed_split_size, int segment_size, int grid_slots, int variant, const int32_t* wg_order,
    float sm_scale, float* part_o, float* part_lse, int part_batch, int part_stride, void* o,
    int workers, void* stream) {
  const char* name = "flash_decode_fp8_fwd";
  SID_REQUIRE(batch >= 0, "%s: negative batch", name);
  SID_REQUIRE(variant >= 0 && variant < kNumVariants, "%s: unknown variant %d", name, variant);
  if (batch == 0) return SID_OK;
  int rc = check_decode_args(name, q, k_cache, v_cache, kv_indptr, kv_indices, o, batch,
                             num_q_heads, num_kv_heads, head_dim, num_slots, max_splits,
                             fixed_split_size);
  if (rc != SID_OK) return rc;
  SID_REQUIRE(kv_scales != nullptr, "%s: null pointer", name);
  auto misaligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  SID_REQUIRE(!misaligned(q) && !misaligned(k_cache) && !misaligned(v_cache) &&
                  !misaligned(kv_scales) && !misaligned(o) && !misaligned(part_o),
              "%s: operands must be 16-byte aligned", name);
  rc = check_decode_plan(name, batch, segment_size, grid_slots, wg_order, workers, part_o,
                         part_lse, part_batch, part_stride);
  if (rc != SID_OK) return rc;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool direct = grid_slots == 1;
  const bool worker = workers > 0 && !direct;
  auto stage1 = [&](auto kern, int nw) {
    hipLaunchKernelGGL(kern, worker ? dim3(workers) : dim3(batch, grid_slots), dim3(nw * 64), 0, s,
                       (const bf16_t*)q, (const uint8_t*)k_cache, (const uint8_t*)v_cache,
                       (const uint16_t*)kv_scales, kv_indptr, kv_indices, num_splits, max_splits,
                       fixed_split_size, segment_size, sm_scale, num_slots, part_stride, part_o,
                       part_lse, direct ? (bf16_t*)o : nullptr, wg_order, batch, grid_slots);
  };
  if (variant == 2) {
    worker ? stage1(decode_fp8_stage1_kernel<8, true>, 8)
           : stage1(decode_fp8_stage1_kernel<8, false>, 8);
  } else {
    worker ? stage1(decode_fp8_stage1_kernel<4, true>, 4)
           : stage1(decode_fp8_stage1_kernel<4, false>, 4);
  }
  rc = check_launch("flash_decode_fp8_fwd stage1");
  if (rc != SID_OK || direct) return rc;
  return launch_decode_stage2(batch, grid_slots, part_o, part_lse, part_stride, o, s);
}
