// Varlen causal "extend" attention over the 8-bit pool (format: kv_fp8.h), gfx950 MFMA.
//
// The contract, the splits, the tile arithmetic and the fan-out are extend_attention.hip's
// (extend_tile.h). Codes become bf16 values on their way into the LDS tiles, exactly, so a
// result has the bits that the bf16 kernels give on the pool read back: independent of the
// window, the batch and the launch's form.
#include "extend_tile.h"
#include "kv_fp8.h"

#include <type_traits>

namespace sid {
namespace {

// ---- staging -------------------------------------------------------------------------------
//
// A tile's K (and V) is 512 pieces of 16 codes: piece p is key p / 8, dims 16 (p % 8) .. +15. A
// thread holds PER pieces of each between the global loads, issued a whole tile ahead, and the
// LDS, where they are two 16-byte pieces of bf16.
template <int PER>
struct Raw {
  u32x4_v k[PER];
  u32x4_v v[PER];
  uint32_t s[PER];  // the key's scale bytes, K | V << 8
};

// A NaN vector must reach the queries that see its key and no others, but a hidden key's value
// is multiplied by p = 0, which leaves a NaN. So a key whose K or V is NaN gets NaN scores (a
// hidden key's scores are never used) and values 0, and a key past the sequence's end (which
// every query hides) values 0. Both are rare: one test finds that a wave has none.
template <int PER>
__device__ __forceinline__ void guard(Raw<PER>& r, int i, bool exists) {
  const bool nan = (r.s[i] & 255u) == kScaleNaN || r.s[i] >> 8 == kScaleNaN;
  if (__builtin_amdgcn_ballot_w64(nan || !exists) == 0) return;
  if (nan) {
    r.k[i] = u32x4_v{kCodesNaN, kCodesNaN, kCodesNaN, kCodesNaN};
    r.s[i] = 127u | 127u << 8;
  }
  if (nan || !exists) r.v[i] = u32x4_v{0, 0, 0, 0};
}

// 16 codes times 2^e as two 16-byte pieces of bf16.
__device__ __forceinline__ void unpack16(u32x4_v c, uint32_t byte, u32x4_v (&out)[2]) {
  const float s = fp8_scale(byte);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint2 a = fp8_to_bf16x4(c[2 * i], s), b = fp8_to_bf16x4(c[2 * i + 1], s);
    out[i] = u32x4_v{a.x, a.y, b.x, b.y};
  }
}

struct RowCtx {  // what softmax_tile reads
  int g;
  int q_abs;
  bool row_ok;
};

// Workgroup = (request, kv head, 8 NW query positions), NW waves; wave w: head w / (NW / 2), one
// block of 16 query rows. FANOUT (NW = 4): the workgroup computes one split and saves its state
// for the fold; else it walks the splits in order.
template <int NW, bool FANOUT>
__global__ void __launch_bounds__(NW * 64, NW / 2) extend_fp8_kernel(
    const bf16_t* __restrict__ q, const uint8_t* __restrict__ k_cache,
    const uint8_t* __restrict__ v_cache, const uint16_t* __restrict__ kv_scales,
    const int32_t* __restrict__ qo_indptr, const int32_t* __restrict__ kv_indptr,
    const int32_t* __restrict__ kv_indices, int batch, int num_q_heads, int num_kv_heads,
    int64_t num_slots, float sm_scale, int mtiles, int64_t items, bf16_t* __restrict__ o,
    float* __restrict__ part_a, float* __restrict__ part_ml, int32_t* __restrict__ part_n) {
  extern __shared__ __align__(1024) char lds[];  // [2][K tile, V tile], bf16
  constexpr int ROWS = 8 * NW;
  constexpr int PER = 8 / NW;
  const int b = min(static_cast<int>(blockIdx.x), batch - 1);
  const int h_kv = blockIdx.y;
  // Late query tiles walk the most keys: dispatch them first.
  const int mtile = FANOUT ? static_cast<int>(blockIdx.z) % mtiles
                           : mtiles - 1 - static_cast<int>(blockIdx.z);
  const int split = FANOUT ? static_cast<int>(blockIdx.z) / mtiles : 0;
  const int q_start = qo_indptr[b];
  const int extend_len = qo_indptr[b + 1] - q_start;
  if (mtile * ROWS >= extend_len || static_cast<int>(blockIdx.x) >= batch) return;
  const int kv_start = kv_indptr[b];
  const int kv_len = kv_indptr[b + 1] - kv_start;
  const int prefix = kv_len - extend_len;
  if (prefix < 0) return;  // malformed batch: the kv range must cover the extend tokens

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int hq = h_kv * 2 + wave / (NW / 2);
  const int w_row = mtile * ROWS + 16 * (wave % (NW / 2));  // the wave's first query row
  const int qr = w_row + (lane & 15);
  const bool row_ok = qr < extend_len;
  const int64_t prow = static_cast<int64_t>(q_start + (row_ok ? qr : 0)) * num_q_heads + hq;
  const float sc2 = sm_scale * LOG2E;
  const int last_row = min(extend_len, (mtile + 1) * ROWS) - 1;
  const int visible_end = min(kv_len, prefix + last_row + 1);
  const int nsplits = ceil_div(visible_end, KSPLIT);
  if (FANOUT && split >= nsplits) return;  // the merge never reads this split
  // Tiles [t_begin, t_end) of the sequence.
  const int t_begin = split * (KSPLIT / BN);
  const int t_end = FANOUT ? min(ceil_div(visible_end, BN), t_begin + KSPLIT / BN)
                           : ceil_div(visible_end, BN);
  const int w_first = prefix + w_row;  // the wave's first and last positions
  const int w_last = prefix + min(extend_len, w_row + 16) - 1;

  bf16x8_v qf[4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    qf[ks] = *reinterpret_cast<const bf16x8_v*>(q + prow * D + 32 * ks + 8 * (lane >> 4));
    if (!row_ok) qf[ks] = bf16x8_v{};
  }

  const int32_t* idx = kv_indices + kv_start;
  const uint32_t max_slots = static_cast<uint32_t>(min<int64_t>(num_slots, 0x7fffffff));
  const uint8_t* kb = k_cache + h_kv * D + 16 * (tid & 7);
  const uint8_t* vb = v_cache + h_kv * D + 16 * (tid & 7);
  const uint16_t* sb = kv_scales + h_kv;
  struct Slots {
    uint32_t s[PER];
  };
  auto load_slots = [&](int tile) {
    Slots v;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int key = tile * BN + ((tid + 64 * NW * i) >> 3);
      v.s[i] = key < kv_len ? idx[key] : 0;
    }
    return v;
  };
  Raw<PER> raw;
  auto load_raw = [&](const Slots& v) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t slot = v.s[i] < max_slots ? v.s[i] : 0u;  // (out of range: slot 0)
      raw.k[i] = *reinterpret_cast<const u32x4_v*>(kb + slot * num_kv_heads * D);
      raw.v[i] = *reinterpret_cast<const u32x4_v*>(vb + slot * num_kv_heads * D);
      raw.s[i] = sb[slot * num_kv_heads];
    }
  };
  auto store_raw = [&](int tile) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int key = (tid + 64 * NW * i) >> 3;
      guard(raw, i, tile * BN + key < kv_len);
      u32x4_v k[2], v[2];
      unpack16(raw.k[i], raw.s[i] & 255u, k);
      unpack16(raw.v[i], raw.s[i] >> 8, v);
      char* dst = lds + (tile & 1) * 2 * kTileBytes + 256 * key;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = 16 * ((2 * (tid & 7) + e) ^ swz(key));
        *reinterpret_cast<u32x4_v*>(dst + at) = k[e];
        *reinterpret_cast<u32x4_v*>(dst + kTileBytes + at) = v[e];
      }
    }
  };

  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char_t)lds));
  RowState run, st;
  fresh(run);
  fresh(st);
  // One tile's math out of LDS buffer `buf`. MASK: some key is hidden from some row.
  auto tile_math = [&](auto mask, int t0, int buf) {
    int l = lane;  // opaque: per-lane constants are not kept in registers between tiles
    asm volatile("" : "+v"(l));
    const int r = l & 15, g = l >> 4;
    const int key_a0 = 8 * (r >> 2) + (r & 3);
    const uint32_t ka = lds0 + buf * 2 * kTileBytes + key_a0 * 256 + 16 * (g ^ swz(key_a0));
    f32x4_v s4[4];
#pragma unroll
    for (int i = 0; i < 16; ++i) {  // key block j, k-step ks
      const int j = i & 3, ks = i >> 2;
      const bf16x8_v kf = *(__attribute__((address_space(3))) const bf16x8_v*)(
          (ka ^ (64u * ks)) + 256 * (32 * (j >> 1) + 4 * (j & 1)));
      s4[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
          kf, qf[ks], ks == 0 ? f32x4_v{0.0f, 0.0f, 0.0f, 0.0f} : s4[j], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    const RowCtx c{g, w_first + r, row_ok};
    float s[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = s4[i >> 2][i & 3];
    const float rescale = softmax_tile<decltype(mask)::value>(s, st, c, t0, sc2);
    bf16x8_v pf[2];
    pack_p(pf, s);
    __builtin_amdgcn_sched_barrier(0);
    apply_rescale(st, rescale);
    const int key_v = 8 * g + (r >> 2);
    const uint32_t va = lds0 + (buf * 2 + 1) * kTileBytes + key_v * 256 +
                        16 * (((r & 3) >> 1) ^ swz(key_v)) + 8 * (r & 1);
#pragma unroll
    for (int i = 0; i < 16; ++i) {  // dim block db, key half kb
      const int db = i & 7, kb2 = i >> 3;
      typedef __attribute__((address_space(3))) s16x4_v* tr_ptr_t;
      const uint32_t p = (va ^ (32u * db)) + 8192 * kb2;
      const s16x4_v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)p);
      const s16x4_v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)(p + 1024));
      const bf16x8_v vf = __builtin_bit_cast(
          bf16x8_v, static_cast<s16x8_v>(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)));
      st.acc[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[kb2], st.acc[db], 0, 0, 0);
    }
  };

  load_raw(load_slots(t_begin));
  Slots next = load_slots(t_begin + 1);
  store_raw(t_begin);
  load_raw(next);
  next = load_slots(t_begin + 2);
  for (int t = t_begin; t < t_end; ++t) {
    __syncthreads();  // tile t is stored and every wave is done with the other buffer
    if (t + 1 < t_end) {
      store_raw(t + 1);
      load_raw(next);
      next = load_slots(t + 3);
    }
    const int t0 = t * BN;
    if (t0 + BN - 1 <= w_first && w_row < extend_len) {
      tile_math(std::false_type{}, t0, t & 1);
    } else if (t0 <= w_last && w_row < extend_len) {
      tile_math(std::true_type{}, t0, t & 1);
    }
    if (!FANOUT && ((t & 3) == 3 || t + 1 == t_end)) {  // the split's end
      fold(run, st.m, st.l, st.acc);
      fresh(st);
    }
  }
  if (!row_ok) return;
  if constexpr (FANOUT) {
    const int64_t pr = split * items + prow;
    const int g = lane >> 4;
#pragma unroll
    for (int db = 0; db < 8; ++db)
      *reinterpret_cast<f32x4_v*>(part_a + pr * D + 16 * db + 4 * g) = st.acc[db];
    if (g == 0) {
      part_ml[2 * pr] = st.m;
      part_ml[2 * pr + 1] = st.l;
      if (split == 0) part_n[prow] = nsplits;
    }
  } else {
    store_row(o + prow * D, run, lane >> 4);
  }
}

}  // namespace
}  // namespace sid

using namespace sid;

extern "C" int sid_extend_attention_fp8_fwd(
    const void* q, const void* k_cache, const void* v_cache, const void* kv_scales,
    const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices, int batch,
    int64_t total_q, int num_q_heads, int num_kv_heads, int head_dim, int64_t num_slots,
    int max_extend_len, int max_kv_len, float sm_scale, void* workspace, int64_t workspace_bytes,
    void* o, void* stream) {
  const char* name = "extend_attention_fp8";
  const ExtendPlan p = extend_plan(name, q, k_cache, v_cache, qo_indptr, kv_indptr, kv_indices, o,
                                   batch, total_q, num_q_heads, num_kv_heads, head_dim, num_slots,
                                   max_extend_len, max_kv_len, workspace, workspace_bytes);
  if (p.rc != SID_OK || p.empty) return p.rc;
  SID_REQUIRE(kv_scales != nullptr, "%s: null pointer", name);
  auto misaligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) != 0; };
  SID_REQUIRE(!misaligned(q) && !misaligned(k_cache) && !misaligned(v_cache) &&
                  !misaligned(kv_scales) && !misaligned(o) && !misaligned(workspace),
              "%s: operands must be 16-byte aligned", name);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto kern, int nw, dim3 grid) {
    hipLaunchKernelGGL(kern, grid, dim3(nw * 64), 4 * kTileBytes, s, (const bf16_t*)q,
                       (const uint8_t*)k_cache, (const uint8_t*)v_cache,
                       (const uint16_t*)kv_scales, qo_indptr, kv_indptr, kv_indices, batch,
                       num_q_heads, num_kv_heads, num_slots, sm_scale, p.mtiles, p.items,
                       (bf16_t*)o, p.part_a, p.part_ml, p.part_n);
    return check_launch(name);
  };
  if (p.fanout) {
    const int rc = launch(extend_fp8_kernel<4, true>, 4,
                          dim3(batch, num_kv_heads, p.mtiles * p.splits));
    return rc != SID_OK ? rc : extend_merge(name, p, o, s);
  }
  const dim3 grid(p.grid_x, num_kv_heads, p.mtiles);
  return p.rows == 64 ? launch(extend_fp8_kernel<8, false>, 8, grid)
                      : launch(extend_fp8_kernel<4, false>, 4, grid);
}
