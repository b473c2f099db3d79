// Varlen causal "extend" attention over the 4-bit pool (format: kv_fp4.h), gfx950 MFMA.
//
// The contract is extend_attention.hip's (a query's result depends only on its position and its
// sequence's keys); the fold of the splits, the fan-out's merge and the placement are shared with the
// other pools' kernels (extend_tile.h, extend_codes.h). The tile arithmetic is this kernel's: K's codes
// lie in the LDS as they are and S = K Q^T is taken on them, a lane's 32 codes with their block's
// scale, with q as two e4m3 vectors; V's become bf16 on their way into the LDS; splits are of 512
// keys.
//
// Rounded to fewer than 32 bits: p, to bf16 before the product with V (half a step, 2^-8 of p, as
// over the other pools: both operands of the product are bf16, and P in two parts would double the
// products), while l sums the unrounded p; and the small elements of a q row that holds far larger
// ones (QRow).
#include "extend_codes.h"
#include "kv_fp4.h"

#include <algorithm>

namespace sid {
namespace {

constexpr int NW = 4;  // waves of a workgroup
constexpr int kSplit = 512;  // keys per split: the unit in which a row's state is folded
constexpr int kSplitTiles = kSplit / BN;

// ---- LDS ---------------------------------------------------------------------------------
//
// A tile is 64 keys. K stays in codes, 64 bytes a key: 16-byte unit u of a key's row holds block
// u ^ swk(key), so that the 16 rows of a fragment read fall on all 64 banks. V is bf16 (swv). Beside
// them K's scale bytes as the matrix instruction takes them: word l holds lane l's for the tile's
// four key blocks.
constexpr int kKTile = BN * D / 2;
constexpr int kVAt = 2 * kKTile;  // [2] K tiles, [2] V tiles, [2] K scale words
constexpr int kScalesAt = kVAt + 2 * kTileBytes;
constexpr int kParkedAt = kScalesAt + 2 * 256;
// The rows' folded state stays in the LDS between two folds, 8 tiles apart: 8 accumulator vectors a
// lane and row set (the registers hold the state of the split in work).
constexpr int lds_bytes(int sets, bool fanout) { return kParkedAt + (fanout ? 0 : 8 * sets * NW * 1024); }

__device__ __forceinline__ int swk(int key) { return (key >> 3) & 3; }

// Workgroup = (request, kv head, 8 NW SETS query positions), NW waves. A wave has SETS sets of 16
// rows: with 2, the two query heads at its 16 positions, which share every K and V fragment that it
// reads; with 1, one head (w / (NW / 2)). FANOUT: the workgroup computes one split and saves its
// state for the fold; else it walks the splits in order.
template <int SETS, bool FANOUT>
__global__ void __launch_bounds__(NW * 64, SETS == 1 ? 2 : 1) extend_fp4_kernel(
    const bf16_t* __restrict__ q, const uint8_t* __restrict__ k_cache,
    const uint8_t* __restrict__ v_cache, const uint2* __restrict__ kv_scales,
    const int32_t* __restrict__ qo_indptr, const int32_t* __restrict__ kv_indptr,
    const int32_t* __restrict__ kv_indices, int batch, int num_q_heads, int num_kv_heads,
    int64_t num_slots, float sm_scale, int mtiles, int per_round, int ordered, int across,
    int64_t items, bf16_t* __restrict__ o, float* __restrict__ part_a,
    float* __restrict__ part_ml, int32_t* __restrict__ part_n) {
  __shared__ __align__(1024) char lds[lds_bytes(SETS, FANOUT)];
  constexpr int ROWS = 8 * NW * SETS;
  int b, h_kv, mtile, split = 0;
  if constexpr (FANOUT) {
    b = blockIdx.x;
    h_kv = blockIdx.y;
    mtile = static_cast<int>(blockIdx.z) % mtiles;
    split = static_cast<int>(blockIdx.z) / mtiles;
  } else {
    // Heads fastest: with 8 of them a head's workgroups, which share its keys, are on one XCD.
    h_kv = blockIdx.x % num_kv_heads;
    const Item it = pick_item<ROWS>(blockIdx.x / num_kv_heads + blockIdx.y * across, ordered != 0,
                                    per_round, batch, mtiles, qo_indptr, kv_indptr);
    if (it.mtile < 0) return;
    b = it.b;
    mtile = it.mtile;
  }
  const int q_start = qo_indptr[b];
  const int extend_len = qo_indptr[b + 1] - q_start;
  if (mtile * ROWS >= extend_len) return;
  const int kv_start = kv_indptr[b];
  const int kv_len = kv_indptr[b + 1] - kv_start;
  const int prefix = kv_len - extend_len;
  if (prefix < 0) {  // malformed batch: the kv range must cover the extend tokens
    if (FANOUT && split == 0)
      skip_rows(part_n, q_start, mtile * ROWS, min(extend_len, (mtile + 1) * ROWS), num_q_heads, h_kv);
    return;
  }

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int hq = h_kv * 2 + (SETS == 2 ? 0 : wave / (NW / 2));  // of set 0
  const int w_row = mtile * ROWS + 16 * (SETS == 2 ? wave : wave % (NW / 2));  // the wave's first query row
  const int r = lane & 15, g = lane >> 4;
  const bool row_ok = w_row + r < extend_len;
  const int64_t prow = static_cast<int64_t>(q_start + (row_ok ? w_row + r : 0)) * num_q_heads + hq;
  const float sc2 = sm_scale * LOG2E;
  const int last_row = min(extend_len, (mtile + 1) * ROWS) - 1;
  const int visible_end = min(kv_len, prefix + last_row + 1);
  const int nsplits = ceil_div(visible_end, kSplit);
  if (FANOUT && split >= nsplits) return;  // the merge never reads this split
  // Tiles [t_begin, t_end) of the sequence.
  const int t_begin = split * kSplitTiles;
  const int t_end = FANOUT ? min(ceil_div(visible_end, BN), t_begin + kSplitTiles)
                           : ceil_div(visible_end, BN);
  const int q_abs = prefix + w_row + r;  // the lane's position
  // The wave's tiles: no row of it sees a key of tile w_tiles or a later one.
  const int w_tiles =
      w_row < extend_len ? (prefix + min(extend_len, w_row + 16) - 1) / BN + 1 : 0;

  // ---- staging. Thread t's piece of 32 codes: key t / 4 of a tile, block t % 4. K's go to the LDS by
  // DMA; V's through registers, where they become bf16 with their scale (once for all waves).
  // During tile t's step K of t + 2 and V of t + 1 load, the scales of t + 3 and the slots of t + 4.
  // No branch guards a load with a register result (past the sequence's end its last key is read
  // again): such a load is waited for where the branch ends, and the tile's DMA with it.
  const int32_t* idx = kv_indices + kv_start;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char_t)lds));
  const uint32_t max_slots = static_cast<uint32_t>(min<int64_t>(num_slots, 0x7fffffff));
  const int my_key = tid >> 2, my_blk = tid & 3;
  auto load_slot = [&](int tile) -> uint32_t { return idx[min(tile * BN + my_key, kv_len - 1)]; };
  // Out of range: slot 0. (Looked at where a slot is used first: at its load, it would be waited
  // for.)
  auto check = [&](uint32_t& slot) { slot = slot < max_slots ? slot : 0; };
  const uint32_t row_bytes = static_cast<uint32_t>(num_kv_heads) * (D / 2);
  const uint8_t* ksrc = k_cache + h_kv * (D / 2) + 16 * (my_blk ^ swk(my_key));
  const uint8_t* vsrc = v_cache + h_kv * (D / 2) + 16 * my_blk;
  const uint2* sbase = kv_scales + h_kv;
  auto load_k = [&](uint32_t slot, int buf) {
    dma16(ksrc + static_cast<uint64_t>(slot) * row_bytes, lds0 + buf * kKTile + 1024u * wave);
  };
  u32x4_v raw;
  auto load_v = [&](uint32_t slot) {
    raw = *reinterpret_cast<const u32x4_v*>(vsrc + static_cast<uint64_t>(slot) * row_bytes);
  };
  auto load_scales = [&](uint32_t slot) {
    return sbase[static_cast<uint64_t>(slot) * static_cast<uint32_t>(num_kv_heads)];
  };
  // This thread's bytes of a head's scales: K | V << 8. A NaN vector must reach the queries that see
  // its key and no others, but a hidden key's value is multiplied by p = 0, which leaves a NaN. So a
  // key whose V is NaN gets a NaN scale for K (E8M0's 255: NaN scores, and a hidden key's scores are
  // never used) and values 0.
  auto my_scales = [&](uint2 s) -> uint32_t {
    const uint32_t k = (s.x >> (8 * my_blk)) & 255u, v = (s.y >> (8 * my_blk)) & 255u;
    return v == kFp4ScaleNaN ? 127u << 8 | kFp4ScaleNaN : v << 8 | k;
  };
  const uint32_t sdst = kScalesAt + 4 * (16 * my_blk + 4 * ((my_key >> 3) & 3) + (my_key & 3)) +
                        2 * (my_key >> 5) + ((my_key >> 2) & 1);
  auto store_scales = [&](uint32_t sc, int buf) {
    reinterpret_cast<uint8_t*>(lds)[sdst + 256 * buf] = static_cast<uint8_t>(sc);
  };
  uint32_t vdst = lds0 + kVAt + 256 * my_key + 16 * ((4 * my_blk) ^ swv(my_key));
  asm volatile("" : "+v"(vdst));
  auto store_v = [&](uint32_t sc, int buf) {
    const bool nan = (sc & 255u) == kFp4ScaleNaN;
    const float s = fp4_scale(sc >> 8);
    typedef __attribute__((address_space(3))) u32x4_v* lds_w_t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 x = fp4_to_bf16x8(nan ? 0u : raw[i], s);
      *(lds_w_t)((vdst ^ (16u * i)) + buf * kTileBytes) = u32x4_v{x.x, x.y, x.z, x.w};
    }
  };

  // The first loads, in the order of their latencies: slots and q, then what the slots name; q is
  // split while those are under way.
  uint32_t sl1 = load_slot(t_begin), sl2 = load_slot(t_begin + 1), sl3 = load_slot(t_begin + 2),
           sl4 = load_slot(t_begin + 3);
  QRaw q_raw[SETS];
#pragma unroll
  for (int s = 0; s < SETS; ++s) q_raw[s] = load_q(q + (prow + s) * D, g);
  __builtin_amdgcn_sched_barrier(0);
  check(sl1);
  check(sl2);
  check(sl3);
  const uint2 s0 = load_scales(sl1), s1 = load_scales(sl2);
  uint2 scales_in = load_scales(sl3);
  load_v(sl1);
  __builtin_amdgcn_sched_barrier(0);
  load_k(sl1, 0);  // (t_begin is a split's first tile: even)
  load_k(sl2, 1);
  __builtin_amdgcn_sched_barrier(0);
  QRow qf[SETS];
#pragma unroll
  for (int s = 0; s < SETS; ++s) qf[s] = split_q(q_raw[s], row_ok);
  __builtin_amdgcn_sched_barrier(0);
  uint32_t sc0 = my_scales(s0), sc1 = my_scales(s1);
  store_scales(sc0, 0);
  store_scales(sc1, 1);
  sl1 = sl2;
  sl2 = sl3;
  sl3 = sl4;
  __builtin_amdgcn_sched_barrier(0);

  // LDS addresses of a lane's fragments in buffer 0, kept in registers.
  // S^T = K Q^T: row m of key block j is key 32 (j / 2) + 8 (m / 4) + 4 (j % 2) + m % 4, so a lane
  // ends with the scores of keys 8 g .. +7 and 32 + 8 g .. +7 of its queries.
  const int key_a0 = 8 * (r >> 2) + (r & 3);
  uint32_t ka = lds0 + key_a0 * (D / 2) + 16 * (g ^ swk(key_a0)), sa = lds0 + kScalesAt + 4 * lane;
  const int key_v = 8 * g + (r >> 2);
  uint32_t va[8];
#pragma unroll
  for (int db = 0; db < 8; ++db) {
    va[db] = (lds0 + kVAt + key_v * 256 + 16 * (((r & 3) >> 1) ^ swv(key_v)) + 8 * (r & 1)) ^ (32u * db);
    asm volatile("" : "+v"(va[db]));
  }
  asm volatile("" : "+v"(ka), "+v"(sa));

  // A step takes the softmax of its tile t between the products of two others: S of tile t + 1 (qk)
  // and the output of tile t - 1 (pv), so that no product waits for this tile's exponentials nor
  // they for it. The softmax is dealt over 8 slices of 2 elements a row set; with them go pv n: key
  // half n / 4, dim blocks 2 (n % 4) and the next; and two slices behind the key block's softmax, as its
  // results take the place of the scores that are used up, qk n: key block n / 2, q's hi part, then
  // its lo part.
  typedef __attribute__((address_space(3))) const u32x4_v* lds_u4_t;
  typedef __attribute__((address_space(3))) s16x4_v* tr_ptr_t;
  u32x4_v kf[2];
  s16x4_v vw[3][2][2];
  f32x4_v s[SETS][4];  // S: row 4 g + i of key block j at [j][i]
  uint4 pn[SETS][2];   // P of this tile, and of the one before
  bf16x8_v pf[SETS][2];
  float m[SETS], l[SETS];  // (l: this lane's 16 keys of every tile)
  f32x4_v acc[SETS][8];
  float run_m[SETS], run_l[SETS];
  typedef __attribute__((address_space(3))) f32x4_v* park_t;
  const park_t parked = (park_t)(lds0 + kParkedAt + 16 * tid);  // vector db of set e: + 64 NW (8 e + db)
#pragma unroll
  for (int e = 0; e < SETS; ++e) {
    m[e] = run_m[e] = NEG_BIG;
    l[e] = run_l[e] = 0.0f;
#pragma unroll
    for (int db = 0; db < 8; ++db) {
      acc[e][db] = f32x4_v{0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (!FANOUT) parked[64 * NW * (8 * e + db)] = acc[e][db];
    }
    pf[e][0] = pf[e][1] = bf16x8_v{};
  }
  auto read_k = [&](auto j_, int buf) {
    constexpr int j = decltype(j_)::value;
    kf[j & 1] = *(lds_u4_t)(ka + buf * kKTile + (32 * (j >> 1) + 4 * (j & 1)) * (D / 2));
  };
  // V fragments: A = V^T rows 16 db + r (dims), columns 32 kb + 8 g .. +7 (keys), by two
  // transpose reads (extend_attention.hip): slice n's, two slices ahead.
  auto read_v = [&](auto n_, int buf) {
    constexpr int n = decltype(n_)::value;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t at = va[2 * (n & 3) + i] + buf * kTileBytes + 8192 * (n >> 2);
      vw[n % 3][i][0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)at);
      vw[n % 3][i][1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)(at + 1024));
    }
  };
  auto qk = [&](auto n_, int e, int ks) {
    constexpr int n = decltype(n_)::value, j = n >> 1;
    constexpr bool lo = (n & 1) != 0;
    const u32x4_v kk = kf[j & 1];
    const i32x8_v a{(int)kk.x, (int)kk.y, (int)kk.z, (int)kk.w, 0, 0, 0, 0};
    // (formats 4 and 0: e2m1 and e4m3; the scale operands' byte is an immediate: key block j of ks,
    // hi or lo of the row's scale)
    if constexpr (lo)
      s[e][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, qf[e].lo, s[e][j], 4, 0, j, ks, 1, qf[e].scale);
    else
      s[e][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
          a, qf[e].hi, f32x4_v{0.0f, 0.0f, 0.0f, 0.0f}, 4, 0, j, ks, 0, qf[e].scale);
  };
  auto pv = [&](auto n_, int i, int e) {
    constexpr int n = decltype(n_)::value;
    const bf16x8_v vf = __builtin_bit_cast(
        bf16x8_v, static_cast<s16x8_v>(__builtin_shufflevector(vw[n % 3][i][0], vw[n % 3][i][1], 0, 1, 2,
                                                               3, 4, 5, 6, 7)));
    f32x4_v& a = acc[e][2 * (n & 3) + i];
    a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[e][n >> 2], a, 0, 0, 0);
  };
  auto each = [](auto f) {  // f(0) .. f(7), as constants
    f(std::integral_constant<int, 0>{}); f(std::integral_constant<int, 1>{});
    f(std::integral_constant<int, 2>{}); f(std::integral_constant<int, 3>{});
    f(std::integral_constant<int, 4>{}); f(std::integral_constant<int, 5>{});
    f(std::integral_constant<int, 6>{}); f(std::integral_constant<int, 7>{});
  };
  typedef std::integral_constant<int, 0> c0;
  auto point = [] { __builtin_amdgcn_sched_barrier(0); };
  // The state (om, ol) and acc of a split that is complete, into the rows'.
  auto fold_split = [&](const float (&om)[SETS], const float (&ol)[SETS]) {
#pragma unroll
    for (int e = 0; e < SETS; ++e) {
      const FoldScale f = fold_scale(run_m[e], om[e]);
      run_l[e] = fold_elem(run_l[e], pair32_sum(pair16_sum(ol[e])), f);
      run_m[e] = f.mn;
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        f32x4_v a = parked[64 * NW * (8 * e + db)];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = fold_elem(a[i], acc[e][db][i], f);
        parked[64 * NW * (8 * e + db)] = a;
      }
    }
  };

  // Tile t's step. MASK: some key of it may be hidden from some row. FIRST: of a split.
  auto step = [&](auto mask, auto first, int t, auto buf) {
    constexpr bool kMask = decltype(mask)::value, kFirst = decltype(first)::value;
    // Every wave is done with the buffers that are written next, and every load has landed (they had a
    // whole tile's time) but V's, the last that went out, which the step's end waits for.
    point();
    asm volatile("s_waitcnt vmcnt(1) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    point();
    const bool mine = !kMask || t <= w_tiles;  // (at w_tiles the tile before is still to be added)
    int ks = 0;
    if (mine) {
      read_v(c0{}, other(buf));
      read_v(std::integral_constant<int, 1>{}, other(buf));
      ks = *(__attribute__((address_space(3))) const int*)(sa + 256 * other(buf));
      read_k(c0{}, other(buf));
    }
    point();
    asm volatile("" : "+v"(scales_in.x), "+v"(scales_in.y));  // (not looked at ahead of the barrier)
    const uint32_t sc2nd = my_scales(scales_in);
    store_scales(sc2nd, buf);
    check(sl3);
    scales_in = load_scales(sl3);
    const uint32_t k_at = sl2, v_at = sl1;
    sl1 = sl2;
    sl2 = sl3;
    sl3 = load_slot(t + 4);
    point();
    if (t + 2 < t_end) load_k(k_at, buf);
    point();
    auto stage_v = [&] {
      asm volatile("" : "+v"(raw));
      store_v(sc0, buf);
      sc0 = sc1;
      sc1 = sc2nd;
      point();
      load_v(v_at);  // last
      point();
    };
    if (!mine) {
      stage_v();
      return;
    }
    float om[SETS], ol[SETS];
    bool vis[16];
    if constexpr (kMask) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        vis[i] = (t * BN + 32 * (i >> 3) + 8 * g + (i & 7) <= q_abs) & row_ok;
    }
    float tmax[SETS];
    bool high = kFirst;
#pragma unroll
    for (int e = 0; e < SETS; ++e) {
      om[e] = m[e];
      ol[e] = l[e];
      if constexpr (kFirst) {
        m[e] = NEG_BIG;
        l[e] = 0.0f;
      }
      tmax[e] = NEG_BIG;
#pragma unroll
      for (int i = 0; i < 16; ++i) tmax[e] = fmaxf(tmax[e], !kMask || vis[i] ? s[e][i >> 2][i & 3] : NEG_BIG);
      high |= tmax[e] * sc2 > m[e] + LAZY_T;
    }
    // Each lane looks at its own scores: only where one of them is LAZY_T above its row's
    // reference maximum (seldom, but for a split's first tile) are the rows' maxima taken.
    const bool moved = kFirst || __builtin_amdgcn_ballot_w64(high) != 0;
    float rescale[SETS];
#pragma unroll
    for (int e = 0; e < SETS; ++e) rescale[e] = 1.0f;
    if (moved) {
#pragma unroll
      for (int e = 0; e < SETS; ++e) {
        const float mc = pair32_max(pair16_max(tmax[e])) * sc2;
        const float m_used = mc > m[e] + LAZY_T ? mc : m[e];
        rescale[e] = exp2_fast(m[e] - m_used);
        m[e] = m_used;
        if constexpr (!kFirst) l[e] *= rescale[e];
      }
    }
    // (One wave has a SIMD to itself: while a product runs, only what follows it in program order can
    // issue, and a second product behind it waits for the first. So between two products stands about
    // as much of the softmax as the first one takes: 34 cycles a qk, 16 a pv, 16 an exponential.)
    each([&](auto n_) {
      constexpr int n = decltype(n_)::value, j = n >> 1, i0 = 2 * (n & 1);
      typedef std::integral_constant<int, n < 2 ? 0 : n - 2> nq;
      float x[SETS][2], p[SETS][2];
      point();
      if constexpr (n < 6) read_v(std::integral_constant<int, n + 2>{}, other(buf));
      if constexpr (n % 2 == 0 && n > 0) read_k(std::integral_constant<int, n / 2>{}, other(buf));
#pragma unroll
      for (int e = 0; e < SETS; ++e)
#pragma unroll
        for (int i = 0; i < 2; ++i) x[e][i] = __builtin_fmaf(s[e][j][i0 + i], sc2, -m[e]);
      point();
      if constexpr (n >= 2) qk(nq{}, 0, ks);
      point();
      p[0][0] = exp2_fast(x[0][0]);
      p[0][1] = exp2_fast(x[0][1]);
      point();
      if constexpr (n >= 2 && SETS == 2) qk(nq{}, 1, ks);
      point();
      if constexpr (SETS == 2) {
        p[1][0] = exp2_fast(x[1][0]);
        p[1][1] = exp2_fast(x[1][1]);
      }
#pragma unroll
      for (int e = 0; e < SETS; ++e) {
        point();
        pv(n_, 0, e);
        point();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (kMask) p[e][i] = vis[2 * n + i] ? p[e][i] : 0.0f;
          l[e] += p[e][i];
        }
        reinterpret_cast<uint32_t*>(&pn[e][n >> 2])[n & 3] = pack_bf16x2(p[e][0], p[e][1]);
      }
#pragma unroll
      for (int e = 0; e < SETS; ++e) {
        point();
        pv(n_, 1, e);
      }
      point();
    });
    // The last key block's products, with V's conversion between them.
    qk(std::integral_constant<int, 6>{}, 0, ks);
    if constexpr (SETS == 2) qk(std::integral_constant<int, 6>{}, 1, ks);
    point();
    stage_v();
    qk(std::integral_constant<int, 7>{}, 0, ks);
    if constexpr (SETS == 2) qk(std::integral_constant<int, 7>{}, 1, ks);
    point();
    // (here, not where the next step uses them: past the branches below they would move there)
#pragma unroll
    for (int e = 0; e < SETS; ++e) {
      asm volatile("" : "+v"(s[e][0]), "+v"(s[e][1]), "+v"(s[e][2]), "+v"(s[e][3]));
      asm volatile("" : "+v"(l[e]), "+v"(pn[e][0].x), "+v"(pn[e][0].y), "+v"(pn[e][0].z), "+v"(pn[e][0].w),
                   "+v"(pn[e][1].x), "+v"(pn[e][1].y), "+v"(pn[e][1].z), "+v"(pn[e][1].w));
    }
    if constexpr (kFirst) {
      if (!FANOUT && t > t_begin) fold_split(om, ol);
#pragma unroll
      for (int e = 0; e < SETS; ++e)
#pragma unroll
        for (int db = 0; db < 8; ++db) acc[e][db] = f32x4_v{0.0f, 0.0f, 0.0f, 0.0f};
    } else if (moved) {  // (x * 1 == x for the rows that did not)
#pragma unroll
      for (int e = 0; e < SETS; ++e)
#pragma unroll
        for (int db = 0; db < 8; ++db)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[e][db][i] *= rescale[e];
    }
#pragma unroll
    for (int e = 0; e < SETS; ++e)
#pragma unroll
      for (int i = 0; i < 2; ++i) pf[e][i] = __builtin_bit_cast(bf16x8_v, pn[e][i]);
  };

  // S of the first tile.
  auto barrier = [&] {
    point();
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    point();
  };
  barrier();
  {
    const int ks = *(__attribute__((address_space(3))) const int*)sa;
    read_k(c0{}, 0);
    each([&](auto n_) {
      constexpr int n = decltype(n_)::value;
      if constexpr (n < 6 && n % 2 == 0) read_k(std::integral_constant<int, n / 2 + 1>{}, 0);
#pragma unroll
      for (int e = 0; e < SETS; ++e) qk(n_, e, ks);
    });
  }
  // Tiles that every row of the workgroup sees whole, in pairs (their buffers' addresses are
  // immediates), then the others with the mask: one loop each, split by split (a branch between
  // the kinds in one loop, or the fold in it, costs a copy of the accumulators each turn).
  const int t_full = (prefix + mtile * ROWS + 1) / BN;
  constexpr std::true_type yes;
  constexpr std::false_type no;
  typedef std::integral_constant<int, 1> c1;
  for (int s0 = t_begin; s0 < t_end; s0 += kSplitTiles) {
    const int s_end = min(s0 + kSplitTiles, t_end), e = min(s_end, t_full);
    int t = s0;
    if (t < e) step(no, yes, t, c0{});
    else step(yes, yes, t, c0{});
    ++t;
    for (; t + 1 < e; t += 2) {
      step(no, no, t, c1{});
      step(no, no, t + 1, c0{});
    }
    if (t < e) step(no, no, t++, c1{});
    for (; t < s_end; ++t) step(yes, no, t, t & 1);
  }
  // The last tile's output. (Its wave skips no P: a wave without that tile has P = 0.)
  barrier();
  {
    const int buf = (t_end - 1) & 1;
    read_v(c0{}, buf);
    each([&](auto n_) {
      constexpr int n = decltype(n_)::value;
      if constexpr (n < 7) read_v(std::integral_constant<int, n + 1>{}, buf);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < SETS; ++e) pv(n_, i, e);
    });
  }
  if constexpr (FANOUT) {
#pragma unroll
    for (int e = 0; e < SETS; ++e) {
      const float sum = pair32_sum(pair16_sum(l[e]));
      if (!row_ok) continue;
      const int64_t pr = split * items + prow + e;
#pragma unroll
      for (int db = 0; db < 8; ++db)
        *reinterpret_cast<f32x4_v*>(part_a + pr * D + 16 * db + 4 * g) = acc[e][db];
      if (g == 0) {
        part_ml[2 * pr] = m[e];
        part_ml[2 * pr + 1] = sum;
        if (split == 0) part_n[prow + e] = nsplits;
      }
    }
  } else {
    fold_split(m, l);
#pragma unroll
    for (int e = 0; e < SETS; ++e)
    {
      RowState run{run_m[e], run_l[e], {}};
#pragma unroll
      for (int db = 0; db < 8; ++db) run.acc[db] = parked[64 * NW * (8 * e + db)];
      if (row_ok) store_row(o + (prow + e) * D, run, g);
    }
  }
}

// Whether a grid of fewer than 512 workgroups fans out: where walking its keys in one workgroup takes
// longer than the launches and the saved states of total_q rows in every split.
bool fans_out(int batch, int64_t total_q, int num_kv_heads, int max_extend_len, int max_kv_len) {
  const int64_t groups = static_cast<int64_t>(batch) * num_kv_heads * ceil_div(max_extend_len, BQ);
  const int64_t states = total_q * ceil_div(max_kv_len, kSplit);
  return groups < 512 && 110 * static_cast<int64_t>(ceil_div(max_kv_len, BN)) > 1200 + states * 85 / 100;
}

}  // namespace
}  // namespace sid

using namespace sid;

extern "C" int64_t sid_extend_attention_fp4_workspace_bytes(int batch, int64_t total_q,
                                                            int num_q_heads, int num_kv_heads,
                                                            int max_extend_len, int max_kv_len) {
  if (batch <= 0 || total_q <= 0 || max_extend_len <= 0 || max_kv_len <= 0) return 0;
  if (!fans_out(batch, total_q, num_kv_heads, max_extend_len, max_kv_len)) return 0;
  // per (split, row, head): 128 accumulator floats + (m, l); per (row, head): split count
  const int64_t splits = ceil_div(max_kv_len, kSplit);
  return (splits * (D + 2) + 1) * total_q * num_q_heads * static_cast<int64_t>(sizeof(float));
}

extern "C" int sid_extend_attention_fp4_fwd(
    const void* q, const void* k_cache, const void* v_cache, const void* kv_scales,
    const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices, int batch,
    int64_t total_q, int num_q_heads, int num_kv_heads, int head_dim, int64_t num_slots,
    int max_extend_len, int max_kv_len, float sm_scale, void* workspace, int64_t workspace_bytes,
    void* o, void* stream) {
  const char* name = "extend_attention_fp4";
  const ExtendPlan p = extend_plan(name, q, k_cache, v_cache, qo_indptr, kv_indptr, kv_indices, o,
                                   batch, total_q, num_q_heads, num_kv_heads, head_dim, num_slots,
                                   max_extend_len, max_kv_len, kSplit,
                                   sid_extend_attention_fp4_workspace_bytes(
                                       batch, total_q, num_q_heads, num_kv_heads, max_extend_len,
                                       max_kv_len),
                                   workspace, workspace_bytes);
  if (p.rc != SID_OK || p.empty) return p.rc;
  SID_REQUIRE(kv_scales != nullptr, "%s: null pointer", name);
  auto misaligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) != 0; };
  SID_REQUIRE(!misaligned(q) && !misaligned(k_cache) && !misaligned(v_cache) &&
                  !misaligned(kv_scales) && !misaligned(o) && !misaligned(workspace),
              "%s: operands must be 16-byte aligned", name);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  // Tiles may differ in their keys: by the lengths, or by prefixes (of which only the longest key
  // list says something here).
  const int ordered = batch > 1 && batch <= 64 * kOrderSteps &&
                      (8 * total_q < 7 * static_cast<int64_t>(batch) * max_extend_len ||
                       max_kv_len > max_extend_len);
  const int per_round = p.rows == 32 ? max(1, cu_count() / num_kv_heads) : 0;
  auto launch = [&](auto kern, dim3 grid, int mtiles, int across) {
    hipLaunchKernelGGL(kern, grid, dim3(NW * 64), 0, s, (const bf16_t*)q, (const uint8_t*)k_cache,
                       (const uint8_t*)v_cache, (const uint2*)kv_scales, qo_indptr, kv_indptr,
                       kv_indices, batch, num_q_heads, num_kv_heads, num_slots, sm_scale, mtiles,
                       per_round, ordered, across, p.items, (bf16_t*)o, p.part_a, p.part_ml, p.part_n);
    return check_launch(name);
  };
  if (p.fanout) {
    const int rc = launch(extend_fp4_kernel<1, true>, dim3(batch, num_kv_heads, p.mtiles * p.splits),
                          p.mtiles, 0);
    return rc != SID_OK ? rc : extend_merge(name, p, qo_indptr, batch, num_q_heads, o, s);
  }
  const int mtiles = ceil_div(max_extend_len, p.rows);
  const int64_t places = static_cast<int64_t>(batch) * mtiles;
  const int across = static_cast<int>(std::min<int64_t>(places, kMaxGridX / num_kv_heads));
  const int64_t down = (places + across - 1) / across;
  SID_REQUIRE(places < (1ll << 30) && down <= 65535, "%s: grid too large", name);
  const dim3 grid(static_cast<unsigned>(across) * num_kv_heads, static_cast<unsigned>(down));
  return p.rows == 64 ? launch(extend_fp4_kernel<2, false>, grid, mtiles, across)
                      : launch(extend_fp4_kernel<1, false>, grid, mtiles, across);
}
