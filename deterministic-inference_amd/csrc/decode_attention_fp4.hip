// Split-KV paged decode attention over the 4-bit pool (format: kv_fp4.h), gfx950.
//
// The partition into splits and segments, the placement orders, the waves' merge and stage 2
// are decode_attention.hip's (decode_split.h); what a wave does with its tokens, 16 at a time, differs:
//   * scores come from the matrix units on the codes as they are: 16 tokens' K of a kv head (a lane:
//     one block of 32 dims with its scale) times q as two e4m3 vectors (q_codes.h), for all 16 query
//     heads, of which the 2 that belong to the kv head are kept. 8 x 2 such products replace the
//     conversions and dot products that took 24 of the vector ALU's 76 instructions a token, and the
//     softmax is one lane's work for (query head, 4 tokens), not that of every lane of a head;
//   * a row of V is 8 heads x 64 bytes of codes: a 16-byte load of a wave is two tokens' rows. Lane l
//     of a half-wave has kv head l / 4 and block l % 4, converted with its power of two (exact) to fp32
//     and summed in fp32, with the weights from the wave's corner of the LDS;
//   * K's next rows are loaded when this iteration's products are done with the registers, V's when its
//     sums are: each has about an iteration's time, at 17 KB a wave under way.
//
// Workgroups are of 4 waves, two to a CU. (8 waves took 1 to 18 % longer in 30 of 31 batches, as their first
// loads and their merge stand alone on a CU: 1 x 1024 tokens 11.3 and 12.2 us, 32 x 2048 21.0 and 22.4.)
// 128 x 4096 tokens 94-109 us by the card (5.3-6.1 TB/s of codes and scales, where a plain read of memory reaches
// 6.0), 64 x 2048 31, 1 x 131072 53, 1 x 1024 11. In fixed splits of 256 tokens (batch_invariant) 128 x 4096
// 126 (stage 1 119, the merge 6) and 24 requests of 150-20001 tokens 69 instead of 62: a split is four iterations
// of a workgroup, beside q's codes, the first loads, the waves' merge and one more partial. What bounds the large ones is memory; the small ones a
// chain of latencies: lengths, slots, rows, the merge in the LDS and the second launch.
#include "decode_split.h"
#include "kv_fp4.h"
#include "q_codes.h"

#include <type_traits>

namespace sid {
namespace {

typedef float f32x4_v __attribute__((ext_vector_type(4)));

constexpr int NW = 4;             // waves of a workgroup
constexpr int WT = 16;            // tokens of a wave iteration
constexpr int PT = WT / 2;        // those of a half-wave's V rows
constexpr int kPRow = WT + 4;     // floats between two heads' weights (16-byte pieces, spread over the banks)
static_assert(NW * 64 == HQ * HEAD_DIM / 8);
constexpr int kScaleRow = 64 + 16;  // bytes between two tokens' scales

// A wave's own corner of the LDS: no other wave reads it.
struct alignas(16) WaveLds {
  float p[HQ][kPRow];
  float rs[HQ];
  uint8_t sc[WT * kScaleRow];
};

__device__ __forceinline__ float pair_sum(float v) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
__device__ __forceinline__ float pair_max(float v) {
  auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
  p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

// What a wave wrote to its corner is there for its other lanes (the LDS serves a wave in order; this
// holds the compiler to it).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The partial attention of request b over partial slot y (a segment of one split), by one
// workgroup of NW waves taking WT tokens per wave iteration. Every exit is workgroup-uniform.
__device__ __forceinline__ void stage1_item(
    Stage1Lds<NW>& sh, WaveLds (&own)[NW], char* q_rows, int b, int y, const bf16_t* __restrict__ q,
    const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
    const uint8_t* __restrict__ kv_scales, const int32_t* __restrict__ kv_indptr,
    const int32_t* __restrict__ kv_indices, const int32_t* __restrict__ num_splits,
    int max_splits, int fixed_split, int seg, float sm_scale, int64_t num_slots, int part_stride,
    float* __restrict__ part_o, float* __restrict__ part_lse, bf16_t* __restrict__ o_direct) {
  constexpr int IT = NW * WT;  // tokens per workgroup iteration
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int r = lane & 15, g = lane >> 4;  // K: token and block; S: query head, tokens 4 g .. +3
  const int half = lane >> 5;              // V: tokens half, 2 + half, ..,
  const int grp = (lane >> 2) & 7;         // kv head
  const int blk = lane & 3;                // and block of 32 dims

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

  // q as codes, by all threads for all waves (250 instructions a wave if each did all).
  const uint4 q_raw = *reinterpret_cast<const uint4*>(q + out_row * HEAD_DIM + 8 * tid);

  WaveLds& mine = own[wave];
  const int32_t* idx = kv_indices + kv_base;
  // Fewer tokens than an iteration takes: an even number for each wave, as a wave's time goes with its
  // tokens.
  if (end - start < IT) {
    const int n = ceil_div(end - start, 2 * NW) * 2;
    start += wave * n;
    end = min(start + n, end);
  } else {
    start += wave * WT;
  }
  int t0 = start;
  const uint32_t max_slots = static_cast<uint32_t>(min<int64_t>(num_slots, 0x7fffffff));
  uint32_t raw, v_slot[PT];  // slots of token r of the next iteration and of this lane's V rows
  u32x4_v k[HKV], v[PT], sc;
  // Positions past the segment's end load its last token again and get weight 0.
  auto load_idx = [&](int t) { raw = idx[min(t + r, end - 1)]; };
  auto from_lane = [](uint32_t x, int l) -> uint32_t { return __builtin_amdgcn_ds_bpermute(4 * l, x); };
  auto row_at = [](const uint8_t* base, uint32_t slot) {  // 512 bytes a slot
    return reinterpret_cast<const u32x4_v*>(base + (static_cast<uint64_t>(slot >> 23) << 32 | slot << 9));
  };
  const uint8_t* k_base = k_cache + 16 * g;
  const uint8_t* v_base = v_cache + 16 * (lane & 31);
  const uint8_t* s_base = kv_scales + 16 * (lane & 3);
  auto load_k = [&] {
    const uint32_t slot = raw < max_slots ? raw : 0u;
    sc = ld16<true>(reinterpret_cast<const u32x4_v*>(s_base + static_cast<uint64_t>(from_lane(slot, lane >> 2)) * 64u));
    const u32x4_v* row = row_at(k_base, slot);
#pragma unroll
    for (int h = 0; h < HKV; ++h) k[h] = ld16<true>(row + 4 * h);
#pragma unroll
    for (int i = 0; i < PT; ++i) v_slot[i] = from_lane(slot, 2 * i + half);
  };
  // V's rows, behind the slots of the tokens at t: those are waited for while V is under way.
  auto load_v = [&](int t) {
    load_idx(t);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < PT; ++i) v[i] = ld16<true>(row_at(v_base, v_slot[i]));
  };
  load_idx(t0);
  load_k();
  load_v(t0 + IT);
  __builtin_amdgcn_sched_barrier(0);
  split_q_row(q_raw, tid & 15, q_rows + (tid >> 4) * kQRow);
  __syncthreads();
  const QRow qf = read_q_row(q_rows + r * kQRow, g);

  float m = NEG_BIG, l = 0.0f;  // of query head r (l: over the lane's tokens)
  float acc[QPK][32];           // query heads 2 grp and 2 grp + 1, over the half's tokens
#pragma unroll
  for (int h = 0; h < QPK; ++h)
#pragma unroll
    for (int d = 0; d < 32; ++d) acc[h][d] = 0.0f;

  // MORE: the next iteration's rows are loaded, K's once this one's are used up, V's likewise.
  auto iterate = [&](auto more) {
    constexpr bool kMore = decltype(more)::value;
    *reinterpret_cast<u32x4_v*>(mine.sc + (lane >> 2) * kScaleRow + 16 * (lane & 3)) = sc;
    wave_sync();
    f32x4_v s;
#pragma unroll
    for (int h = 0; h < HKV; ++h) {
      const i32x8_v a{(int)k[h].x, (int)k[h].y, (int)k[h].z, (int)k[h].w, 0, 0, 0, 0};
      const int ks = mine.sc[r * kScaleRow + 8 * h + g];
      // (formats 4 and 0: e2m1 and e4m3; the last operands name the scales' bytes)
      f32x4_v d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, qf.hi, f32x4_v{}, 4, 0, 0, ks, 0, qf.scale);
      d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, qf.lo, d, 4, 0, 0, ks, 1, qf.scale);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = h == 0 || (r >> 1) == h ? d[i] : s[i];
    }
    float vs[PT];
#pragma unroll
    for (int i = 0; i < PT; ++i)
      vs[i] = fp4_scale(mine.sc[(2 * i + half) * kScaleRow + 8 * grp + 4 + blk]);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (kMore) load_k();
    __builtin_amdgcn_sched_barrier(0);
    float tmax = NEG_BIG;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = s[i] * sm_scale;
      tmax = t0 + 4 * g + i < end ? fmaxf(tmax, s[i]) : tmax;
    }
    const float mn = fmaxf(m, pair_max(tmax));
    const float rs = __expf(m - mn);
    f32x4_v p;
    float psum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = t0 + 4 * g + i < end ? __expf(s[i] - mn) : 0.0f;
      psum += p[i];
    }
    l = l * rs + psum;
    m = mn;
    // (tokens 0, 2, .., 1, 3, ..: a half's weights in two pieces)
    *reinterpret_cast<f32x2_fp4*>(&mine.p[r][2 * g]) = f32x2_fp4{p[0], p[2]};
    *reinterpret_cast<f32x2_fp4*>(&mine.p[r][PT + 2 * g]) = f32x2_fp4{p[1], p[3]};
    const bool moved = __builtin_amdgcn_ballot_w64(rs != 1.0f) != 0;
    if (moved) {
      if (g == 0) mine.rs[r] = rs;
      wave_sync();
#pragma unroll
      for (int h = 0; h < QPK; ++h) {
        const float x = mine.rs[QPK * grp + h];
#pragma unroll
        for (int d = 0; d < 32; ++d) acc[h][d] *= x;
      }
    }
    wave_sync();
    f32x4_v w[QPK][PT / 4];
#pragma unroll
    for (int h = 0; h < QPK; ++h)
#pragma unroll
      for (int i = 0; i < PT / 4; ++i)
        w[h][i] = *reinterpret_cast<const f32x4_v*>(&mine.p[QPK * grp + h][PT * half + 4 * i]);
#pragma unroll
    for (int t = 0; t < PT; ++t) {
      if (!kMore && t0 + 2 * t >= end) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x2_fp4 x[4];
        x[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[t][i], vs[t], 0);
        x[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[t][i], vs[t], 1);
        x[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[t][i], vs[t], 2);
        x[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[t][i], vs[t], 3);
#pragma unroll
        for (int h = 0; h < QPK; ++h) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            acc[h][8 * i + 2 * e] += w[h][t / 4][t % 4] * x[e].x;
            acc[h][8 * i + 2 * e + 1] += w[h][t / 4][t % 4] * x[e].y;
          }
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (kMore) load_v(t0 + 2 * IT);
    wave_sync();
  };
  // (a wave whose first token is past the segment's end adds nothing)
  for (; t0 < end - IT; t0 += IT) iterate(std::true_type{});
  if (t0 < end) iterate(std::false_type{});

  l = pair_sum(l);
  if (g == 0) {
    sh.m[wave][r] = m;
    sh.l[wave][r] = l;
  }
  // The halves' sums; half h gets and writes query head h of the pair.
#pragma unroll
  for (int d = 0; d < 32; ++d) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[0][d]), __float_as_uint(acc[1][d]),
                                                    false, false);
    acc[0][d] = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<float4*>(&sh.acc[wave][QPK * grp + half][32 * blk + 4 * j]) =
        make_float4(acc[0][4 * j], acc[0][4 * j + 1], acc[0][4 * j + 2], acc[0][4 * j + 3]);
  __syncthreads();
  stage1_merge<NW>(sh, tid, out_row, y, part_stride, part_o, part_lse, o_direct);
}

// Grid form and worker form, as in decode_attention.hip: workgroup (b, y), or the entry of
// wg_order at its linear id; or the items that wg_order deals to each of `gridDim.x` workers
// (order entries i, i + workers, ...; from the first one flagged empty on, all are).
template <bool WORKER>
__global__ void __launch_bounds__(NW * 64, 2) decode_fp4_stage1_kernel(
    const bf16_t* __restrict__ q, const uint8_t* __restrict__ k_cache,
    const uint8_t* __restrict__ v_cache, const uint8_t* __restrict__ kv_scales,
    const int32_t* __restrict__ kv_indptr, const int32_t* __restrict__ kv_indices,
    const int32_t* __restrict__ num_splits, int max_splits, int fixed_split, int seg,
    float sm_scale, int64_t num_slots, int part_stride, float* __restrict__ part_o,
    float* __restrict__ part_lse, bf16_t* __restrict__ o_direct,
    const int32_t* __restrict__ wg_order, int batch, int grid_slots) {
  __shared__ Stage1Lds<NW> sh;
  __shared__ WaveLds own[NW];
  __shared__ __align__(16) char q_rows[HQ * kQRow];
  auto item = [&](int b, int y) {
    stage1_item(sh, own, q_rows, b, y, q, k_cache, v_cache, kv_scales, kv_indptr, kv_indices, num_splits,
                    max_splits, fixed_split, seg, sm_scale, num_slots, part_stride, part_o, part_lse,
                    o_direct);
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

constexpr int kNumVariants = 4;  // the other pools' shapes; here all are the one

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
  auto stage1 = [&](auto kern) {
    hipLaunchKernelGGL(kern, worker ? dim3(workers) : dim3(batch, grid_slots), dim3(NW * 64), 0, s,
                       (const bf16_t*)q, (const uint8_t*)k_cache, (const uint8_t*)v_cache,
                       (const uint8_t*)kv_scales, kv_indptr, kv_indices, num_splits, max_splits,
                       fixed_split_size, segment_size, sm_scale, num_slots, part_stride, part_o,
                       part_lse, direct ? (bf16_t*)o : nullptr, wg_order, batch, grid_slots);
  };
  worker ? stage1(decode_fp4_stage1_kernel<true>) : stage1(decode_fp4_stage1_kernel<false>);
  rc = check_launch("flash_decode_fp4_fwd stage1");
  if (rc != SID_OK || direct) return rc;
  return launch_decode_stage2(batch, grid_slots, part_o, part_lse, part_stride, o, s);
}
