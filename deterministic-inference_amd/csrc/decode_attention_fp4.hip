// Split-KV paged decode attention over the 4-bit pool (format: kv_fp4.h), gfx950.
//
// The partition into splits and segments, the placement orders, the waves' merge and stage 2
// are decode_attention.hip's (decode_split.h); what a wave does with the tokens' rows differs:
//   * a row of K (V) is 8 heads x 64 bytes of codes: one 16-byte load of a wave is the rows of two
//     tokens. Each half of the wave has one of them: lane l of it kv head l / 4 and block l % 4, 32
//     dims with one scale; the scales of (token, head) come as one 8-byte load;
//   * codes are converted with their power of two (exact): K to bf16 pairs for dot products with
//     q, V to fp32.
// The halves' softmax states are merged once, before the waves'.
#include "decode_split.h"
#include "kv_fp4.h"

namespace sid {
namespace {

__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_v, a),
                                         __builtin_bit_cast(bf16x2_v, b), c, false);
}

constexpr int TPL = 4;  // tokens of a lane per wave iteration (a wave: 8)

struct TileRegs {
  u32x4_v k[TPL];
  u32x4_v v[TPL];
  uint2 sc[TPL];
};

// The partial attention of request b over partial slot y (a segment of one split), by one
// workgroup of NW waves taking 2 TPL tokens per wave iteration. Every exit is workgroup-uniform.
template <int NW>
__device__ __forceinline__ void stage1_item(
    Stage1Lds<NW>& sh, int b, int y, const bf16_t* __restrict__ q,
    const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
    const uint2* __restrict__ kv_scales, const int32_t* __restrict__ kv_indptr,
    const int32_t* __restrict__ kv_indices, const int32_t* __restrict__ num_splits,
    int max_splits, int fixed_split, int seg, float sm_scale, int64_t num_slots, int part_stride,
    float* __restrict__ part_o, float* __restrict__ part_lse, bf16_t* __restrict__ o_direct) {
  constexpr int IT = NW * 2 * TPL;  // tokens per workgroup iteration
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int half = lane >> 5;
  const int grp = (lane >> 2) & 7;  // kv head
  const int blk = lane & 3;         // block of 32 dims

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

  // Query heads 2 grp and 2 grp + 1: the lane's 32 dims, packed bf16.
  u32x4_v qv[QPK][4];
#pragma unroll
  for (int h = 0; h < QPK; ++h) {
    const u32x4_v* qb =
        reinterpret_cast<const u32x4_v*>(q + (out_row + QPK * grp + h) * HEAD_DIM + 32 * blk);
#pragma unroll
    for (int i = 0; i < 4; ++i) qv[h][i] = qb[i];
  }
  float m[QPK], l[QPK], acc[QPK][32];
#pragma unroll
  for (int h = 0; h < QPK; ++h) {
    m[h] = NEG_BIG;
    l[h] = 0.0f;
#pragma unroll
    for (int d = 0; d < 32; ++d) acc[h][d] = 0.0f;
  }

  const int32_t* idx = kv_indices + kv_base;
  auto load_idx = [&](int t0, int32_t (&raw)[TPL]) {
#pragma unroll
    for (int t = 0; t < TPL; ++t) raw[t] = idx[min(t0 + 2 * t + half, end - 1)];
  };
  // Positions past the segment's end load its last token again and get weight 0.
  auto load_tile = [&](int t0, const int32_t (&raw)[TPL], bool (&ok)[TPL], TileRegs& r) {
#pragma unroll
    for (int t = 0; t < TPL; ++t) {
      int64_t sv = static_cast<int64_t>(raw[t]);
      if (sv < 0 || sv >= num_slots) sv = 0;
      ok[t] = t0 + 2 * t + half < end;
      r.k[t] = ld16<true>(reinterpret_cast<const u32x4_v*>(k_cache + sv * (HKV * HEAD_DIM / 2)) +
                          (lane & 31));
      r.v[t] = ld16<true>(reinterpret_cast<const u32x4_v*>(v_cache + sv * (HKV * HEAD_DIM / 2)) +
                          (lane & 31));
      r.sc[t] = kv_scales[sv * HKV + grp];
    }
    __builtin_amdgcn_sched_barrier(0);  // (as in decode_attention.hip: all loads go out first)
  };
  auto compute = [&](const bool (&ok)[TPL], const TileRegs& r) {
    float sc[QPK][TPL];
#pragma unroll
    for (int t = 0; t < TPL; ++t) {
      const float ks = fp4_scale((r.sc[t].x >> (8 * blk)) & 255u);
      float s[QPK] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 kc = fp4_to_bf16x8(r.k[t][i], ks);
#pragma unroll
        for (int h = 0; h < QPK; ++h) {
          s[h] = dot2(qv[h][i].x, kc.x, s[h]);
          s[h] = dot2(qv[h][i].y, kc.y, s[h]);
          s[h] = dot2(qv[h][i].z, kc.z, s[h]);
          s[h] = dot2(qv[h][i].w, kc.w, s[h]);
        }
      }
#pragma unroll
      for (int h = 0; h < QPK; ++h) {  // over the head's 4 lanes
        s[h] += dpp<DPP_QUAD_XOR1>(s[h]);
        s[h] += dpp<DPP_QUAD_XOR2>(s[h]);
        sc[h][t] = s[h] * sm_scale;
      }
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
        for (int d = 0; d < 32; ++d) acc[h][d] *= rs;
      }
    }
#pragma unroll
    for (int t = 0; t < TPL; ++t) {
      const float vs = fp4_scale((r.sc[t].y >> (8 * blk)) & 255u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x2_fp4 x[4];
        x[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r.v[t][i], vs, 0);
        x[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r.v[t][i], vs, 1);
        x[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r.v[t][i], vs, 2);
        x[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r.v[t][i], vs, 3);
#pragma unroll
        for (int h = 0; h < QPK; ++h) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[h][8 * i + 2 * e] += sc[h][t] * x[e].x;
            acc[h][8 * i + 2 * e + 1] += sc[h][t] * x[e].y;
          }
        }
      }
    }
  };

  // Rows are loaded one iteration ahead of their math, their slots two.
  int32_t raw[TPL];
  TileRegs r;
  bool ok[TPL];
  int t0 = start + wave * 2 * TPL;
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

  // The halves' states into one: both lanes of a pair compute it on the same operands.
#pragma unroll
  for (int h = 0; h < QPK; ++h) {
    auto pair = [](float v) {
      return __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    };
    const auto pm = pair(m[h]), pl = pair(l[h]);
    const float m0 = __uint_as_float(pm[0]), m1 = __uint_as_float(pm[1]);
    const float mn = fmaxf(m0, m1);
    const float a0 = __expf(m0 - mn), a1 = __expf(m1 - mn);
    m[h] = mn;
    l[h] = __uint_as_float(pl[0]) * a0 + __uint_as_float(pl[1]) * a1;
#pragma unroll
    for (int d = 0; d < 32; ++d) {
      const auto p = pair(acc[h][d]);
      acc[h][d] = __uint_as_float(p[0]) * a0 + __uint_as_float(p[1]) * a1;
    }
    // half h writes query head h of the pair
    if (half == h) {
      const int hq = QPK * grp + h;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        *reinterpret_cast<float4*>(&sh.acc[wave][hq][32 * blk + 4 * j]) =
            make_float4(acc[h][4 * j], acc[h][4 * j + 1], acc[h][4 * j + 2], acc[h][4 * j + 3]);
      if (blk == 0) {
        sh.m[wave][hq] = m[h];
        sh.l[wave][hq] = l[h];
      }
    }
  }
  __syncthreads();
  stage1_merge<NW>(sh, tid, out_row, y, part_stride, part_o, part_lse, o_direct);
}

// Grid form and worker form, as in decode_attention.hip: workgroup (b, y), or the entry of
// wg_order at its linear id; or the items that wg_order deals to each of `gridDim.x` workers
// (order entries i, i + workers, ...; from the first one flagged empty on, all are).
template <int NW, bool WORKER>
__global__ void __launch_bounds__(NW * 64) decode_fp4_stage1_kernel(
    const bf16_t* __restrict__ q, const uint8_t* __restrict__ k_cache,
    const uint8_t* __restrict__ v_cache, const uint2* __restrict__ kv_scales,
    const int32_t* __restrict__ kv_indptr, const int32_t* __restrict__ kv_indices,
    const int32_t* __restrict__ num_splits, int max_splits, int fixed_split, int seg,
    float sm_scale, int64_t num_slots, int part_stride, float* __restrict__ part_o,
    float* __restrict__ part_lse, bf16_t* __restrict__ o_direct,
    const int32_t* __restrict__ wg_order, int batch, int grid_slots) {
  __shared__ Stage1Lds<NW> sh;
  auto item = [&](int b, int y) {
    stage1_item<NW>(sh, b, y, q, k_cache, v_cache, kv_scales, kv_indptr, kv_indices, num_splits,
                    max_splits, fixed_split, seg, sm_scale, num_slots, part_stride, part_o, part_lse,
                    o_direct);
  };
  constexpr int kSlotMask = (1 << kOrderSlotBits) - 1;
  if constexpr (!WORKER) {
    int b = blockIdx.x;
    int y = blockIdx.y;
    if (wg_order != nullptr) {
      const int packed = wg_order[blockIdx.x + blockIdx.y * gridDim.x] & ~kOrderEmpty;
      b = packed >> kOrderSlotBits;
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
      const int b = packed >> kOrderSlotBits;
      const int y = packed & kSlotMask;
      if (b < batch && y < grid_slots) item(b, y);
      __syncthreads();  // the item's merge reads of the LDS are done before the next one's writes
    }
    const int rest = i < n_items ? (n_items - i + W - 1) / W : 0;
    for (int t = threadIdx.x; t < rest * HQ; t += NW * 64) {
      const int packed = wg_order[i + (t / HQ) * W] & ~kOrderEmpty;
      const int b = packed >> kOrderSlotBits;
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

extern "C" int sid_flash_decode_fp4_fwd(
    const void* q, const void* k_cache, const void* v_cache, const void* kv_scales,
    const int32_t* kv_indptr, const int32_t* kv_indices, const int32_t* num_splits, int batch,
    int num_q_heads, int num_kv_heads, int head_dim, int64_t num_slots, int max_splits,
    int fixed_split_size, int segment_size, int grid_slots, int variant, const int32_t* wg_order,
    float sm_scale, float* part_o, float* part_lse, int part_batch, int part_stride, void* o,
    int workers, void* stream) {
  const char* name = "flash_decode_fp4_fwd";
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
                       (const uint2*)kv_scales, kv_indptr, kv_indices, num_splits, max_splits,
                       fixed_split_size, segment_size, sm_scale, num_slots, part_stride, part_o,
                       part_lse, direct ? (bf16_t*)o : nullptr, wg_order, batch, grid_slots);
  };
  if (variant == 2) {
    worker ? stage1(decode_fp4_stage1_kernel<8, true>, 8)
           : stage1(decode_fp4_stage1_kernel<8, false>, 8);
  } else {
    worker ? stage1(decode_fp4_stage1_kernel<4, true>, 4)
           : stage1(decode_fp4_stage1_kernel<4, false>, 4);
  }
  rc = check_launch("flash_decode_fp4_fwd stage1");
  if (rc != SID_OK || direct) return rc;
  return launch_decode_stage2(batch, grid_slots, part_o, part_lse, part_stride, o, s);
}
