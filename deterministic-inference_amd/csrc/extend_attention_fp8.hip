// Varlen causal "extend" attention over the 8-bit pool (format: kv_fp8.h), gfx950 MFMA.
//
// The contract is extend_attention.hip's (a query's result depends only on its position and its
// sequence's keys), and the fold of the splits and the fan-out's merge are shared with it
// (extend_tile.h). The tile arithmetic is this kernel's: K's codes lie in the LDS as they are and S
// = K Q^T is taken on them, with q as two e4m3 vectors; V's become bf16 on their way into the LDS;
// splits are of 512 keys.
//
// Rounded to fewer than 32 bits: p, to bf16 before the product with V (half a step, 2^-8 of p, as
// over the bf16 pool and in sid/kernels/extend_attention.py:106: both operands of the product are
// bf16, and P in two parts would double the products), while l sums the unrounded p; and the small
// elements of a q row that holds far larger ones (QRow). Against 64 bits the result's error, most of
// it the rounding of the result itself, is 8% (ragged chunks) to 15% (4 x 2048 tokens) above that of
// fp32 arithmetic rounded once.
//
// Bound: 4 operations for each of a query's keys and dims. Calls in a row take, for 1 x 8192 tokens,
// 319 us, 0.86 PFLOP/s; for 4 x 2048 102 us, 0.67, a third of which is the workgroups' first loads
// and last stores (one of 8 waves fills a CU; a launch alone takes 120). The 2-byte pool's kernel
// takes 1.19 and 1.08 times as long, 1.5 times on ragged chunks over long prefixes, and 0.93 on
// 16 x 512 tokens and on windows of 32. The matrix products are 1024 of a tile's 2800 cycles on a
// SIMD (two waves, 24 products each); the rest is a wave's own chain, V's conversion, the softmax and
// the loads' addresses, which two waves that start a tile at the same barrier overlap only in part.
// It is not the LDS (896 cycles a tile of 8 waves, no bank conflicts) nor the count of vector
// operations (a third fewer: 2%).
#include "extend_codes.h"

#include <algorithm>

namespace sid {
namespace {

// Keys per split: the unit in which a row's state is folded, and in which a small grid fans out. (256,
// as for bf16 pools: 16 windows of 32 over 2048 keys 47 us against 38, 700 tokens over 4000 99
// against 78; 4 windows 21.1 against 22.5.)
constexpr int kSplit = 512;
constexpr int kSplitTiles = kSplit / BN;

// ---- LDS ---------------------------------------------------------------------------------
//
// A tile is 64 keys. K stays in codes, 128 bytes a key: 16-byte unit u of a key's row holds piece
// u ^ swk(key), so that the 16 rows of a fragment read fall on all 64 banks. V is bf16, 256
// bytes a key, piece p at p ^ swv(key): half a wave's transpose read takes 32 bytes of 8 keys, which
// swv puts on all banks. Beside them K's scale bytes as the matrix instruction takes them: word r
// holds the bytes of row r of the tile's four key blocks.
constexpr int kKTile = BN * D;
constexpr int kVAt = 2 * kKTile;                 // [2] K tiles, [2] V tiles, [2] K scale words
constexpr int kScalesAt = kVAt + 2 * kTileBytes;
constexpr int kParkedAt = kScalesAt + 2 * 64;
// A lane's folded state stays in the LDS between two folds, 8 tiles apart: 7 of its 8
// accumulator vectors (the registers hold the state of the split in work; with all 8, two 4-wave
// workgroups would not fit a CU).
constexpr int kParked = 7;
constexpr int lds_bytes(int waves, bool fanout) {
  return kParkedAt + (fanout ? 0 : kParked * waves * 1024);
}

__device__ __forceinline__ int swk(int key) { return ((key >> 1) & 1) | (((key >> 3) & 3) << 1); }

// 16 codes times 2^e as two 16-byte pieces of bf16.
__device__ __forceinline__ void unpack16(u32x4_v c, uint32_t byte, u32x4_v (&out)[2]) {
  const float s = fp8_scale(byte);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint2 a = fp8_to_bf16x4(c[2 * i], s), b = fp8_to_bf16x4(c[2 * i + 1], s);
    out[i] = u32x4_v{a.x, a.y, b.x, b.y};
  }
}

// Workgroup = (request, kv head, 8 NW query positions), NW waves; wave w: 16 positions of query head
// w / (NW / 2). FANOUT: the workgroup computes one split and saves its state for the fold; else it
// walks the splits in order.
template <int NW, bool FANOUT>
__global__ void __launch_bounds__(NW * 64, 2) extend_fp8_kernel(
    const bf16_t* __restrict__ q, const uint8_t* __restrict__ k_cache,
    const uint8_t* __restrict__ v_cache, const uint16_t* __restrict__ kv_scales,
    const int32_t* __restrict__ qo_indptr, const int32_t* __restrict__ kv_indptr,
    const int32_t* __restrict__ kv_indices, int batch, int num_q_heads, int num_kv_heads,
    int64_t num_slots, float sm_scale, int mtiles, int per_round, int ordered, int across,
    int64_t items, bf16_t* __restrict__ o, float* __restrict__ part_a,
    float* __restrict__ part_ml, int32_t* __restrict__ part_n) {
  __shared__ __align__(1024) char lds[lds_bytes(NW, FANOUT)];
  constexpr int ROWS = 8 * NW;
  int b, h_kv, mtile, split = 0;
  if constexpr (FANOUT) {
    b = blockIdx.x;
    h_kv = blockIdx.y;
    mtile = static_cast<int>(blockIdx.z) % mtiles;
    split = static_cast<int>(blockIdx.z) / mtiles;
  } else {
    // Heads fastest: with 8 of them a head's workgroups, which share its keys, are on one XCD.
    // A grid's first dimension holds `across` places, its second the rows of them (pick_item has
    // no tile for those past the last).
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
  const int hq = h_kv * 2 + wave / (NW / 2);
  const int w_row = mtile * ROWS + 16 * (wave % (NW / 2));  // the wave's first query row
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

  // ---- staging. Thread t's pieces i of 16 codes: key t / 8 + 8 NW i, piece t % 8. K's go to the
  // LDS by DMA; V's through registers, where they become bf16 with their scale (once for all
  // waves: converted at every fragment read instead, 64 more conversions and 32 products a wave
  // and tile). During tile t's step K of t + 2 and V of t + 1 load, the scales of t + 3 and the
  // slots of t + 4. No branch guards a load with a register result (past the sequence's end its
  // last key is read again): such a load is waited for where the branch ends, and the tile's DMA
  // with it.
  constexpr int KP = 8 / NW;
  const int32_t* idx = kv_indices + kv_start;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char_t)lds));
  const uint32_t max_slots = static_cast<uint32_t>(min<int64_t>(num_slots, 0x7fffffff));
  const uint8_t* kb = k_cache + h_kv * D;
  const uint8_t* vb = v_cache + h_kv * D;
  const uint16_t* sb = kv_scales + h_kv;
  struct PerKey {
    uint32_t x[KP];
  };
  auto load_slots = [&](int tile) {
    PerKey v;
#pragma unroll
    for (int i = 0; i < KP; ++i)
      v.x[i] = idx[min(tile * BN + (tid >> 3) + 8 * NW * i, kv_len - 1)];
    return v;
  };
  // Out of range: slot 0. (Looked at where a slot is used first: at its load, it would be waited
  // for.)
  auto check = [&](PerKey& slot) {
#pragma unroll
    for (int i = 0; i < KP; ++i) slot.x[i] = slot.x[i] < max_slots ? slot.x[i] : 0;
  };
  const uint32_t row_bytes = static_cast<uint32_t>(num_kv_heads) * D;
  // (A thread's key of piece i is 8 NW i after its first, a multiple of 32: the swizzles are the same.)
  const uint8_t* ksrc = kb + 16 * ((tid & 7) ^ swk(tid >> 3));
  const uint8_t* vsrc = vb + 16 * (tid & 7);
  auto load_k = [&](const PerKey& slot, int buf) {
#pragma unroll
    for (int i = 0; i < KP; ++i)
      dma16(ksrc + static_cast<uint64_t>(slot.x[i]) * row_bytes,
            lds0 + buf * kKTile + 1024u * (wave + NW * i));
  };
  u32x4_v raw[KP];
  auto load_v = [&](const PerKey& slot) {
#pragma unroll
    for (int i = 0; i < KP; ++i)
      raw[i] = *reinterpret_cast<const u32x4_v*>(vsrc + static_cast<uint64_t>(slot.x[i]) * row_bytes);
  };
  auto load_scales = [&](const PerKey& slot) {  // K | V << 8
    PerKey v;
#pragma unroll
    for (int i = 0; i < KP; ++i) 
      v.x[i] = sb[static_cast<uint64_t>(slot.x[i]) * static_cast<uint32_t>(num_kv_heads)];
    return v;
  };
  // A NaN vector must reach the queries that see its key and no others, but a hidden key's value
  // is multiplied by p = 0, which leaves a NaN. So a key whose K or V is NaN gets a NaN scale for K
  // (E8M0's 255: NaN scores, and a hidden key's scores are never used) and values 0. (Branches
  // would cost more than they skip.)
  auto store_scales = [&](PerKey& sc, auto buf) {
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      sc.x[i] = sc.x[i] >= kScaleNaN << 8 ? 127 << 8 | kScaleNaN : sc.x[i];
      const int key = (tid >> 3) + 8 * NW * i;
      const int m = 4 * ((key >> 3) & 3) + (key & 3), j = 2 * (key >> 5) + ((key >> 2) & 1);
      reinterpret_cast<uint8_t*>(lds + kScalesAt + buf * 64)[4 * m + j] =
          static_cast<uint8_t>(sc.x[i]);
    }
  };
  // Of a key's 8 threads the last 4 write their second piece first: 8 threads write 128 bytes a
  // cycle, which have to lie on different banks.
  const int v_swap = (tid >> 2) & 1;
  uint32_t vdst = lds0 + kVAt + 256 * (tid >> 3) + 16 * ((2 * (tid & 7) + v_swap) ^ swv(tid >> 3));
  asm volatile("" : "+v"(vdst));
  auto store_v = [&](const PerKey& sc, auto buf) {
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const bool nan = (sc.x[i] & 255u) == kScaleNaN;
      u32x4_v c = v_swap ? u32x4_v{raw[i].z, raw[i].w, raw[i].x, raw[i].y} : raw[i];
      c = nan ? u32x4_v{0, 0, 0, 0} : c;
      u32x4_v v[2];
      unpack16(c, sc.x[i] >> 8, v);
      typedef __attribute__((address_space(3))) u32x4_v* lds_w_t;
      *(lds_w_t)(vdst + buf * kTileBytes + 256 * 8 * NW * i) = v[0];
      *(lds_w_t)((vdst ^ 16u) + buf * kTileBytes + 256 * 8 * NW * i) = v[1];
    }
  };

  // The first loads, in the order of their latencies: slots and q, then what the slots name; q is
  // split while those are under way.
  PerKey sl1 = load_slots(t_begin), sl2 = load_slots(t_begin + 1), sl3 = load_slots(t_begin + 2),
         sl4 = load_slots(t_begin + 3);
  const QRaw q_raw = load_q(q + prow * D, g);
  __builtin_amdgcn_sched_barrier(0);
  check(sl1);
  check(sl2);
  check(sl3);
  PerKey sc0 = load_scales(sl1), sc1 = load_scales(sl2), scales_in = load_scales(sl3);
  load_v(sl1);
  __builtin_amdgcn_sched_barrier(0);
  load_k(sl1, 0);  // (t_begin is a split's first tile: even)
  load_k(sl2, 1);
  __builtin_amdgcn_sched_barrier(0);
  const QRow qf = split_q(q_raw, row_ok);
  __builtin_amdgcn_sched_barrier(0);
  store_scales(sc0, 0);
  store_scales(sc1, 1);
  sl1 = sl2;
  sl2 = sl3;
  sl3 = sl4;
  __builtin_amdgcn_sched_barrier(0);

  // LDS addresses of a lane's fragments in buffer 0, kept in registers.
  // S^T = K Q^T: row m of key block j is key 32 (j / 2) + 8 (m / 4) + 4 (j % 2) + m % 4, so a lane
  // ends with the scores of keys 8 g .. +7 and 32 + 8 g .. +7 of its query.
  const int key_a0 = 8 * (r >> 2) + (r & 3);
  uint32_t ka[2], va[8], sa = lds0 + kScalesAt + 4 * r;
#pragma unroll
  for (int e = 0; e < 2; ++e) ka[e] = lds0 + key_a0 * D + 16 * ((g + 4 * e) ^ swk(key_a0));
  const int key_v = 8 * g + (r >> 2);
#pragma unroll
  for (int db = 0; db < 8; ++db)
    va[db] = (lds0 + kVAt + key_v * 256 + 16 * (((r & 3) >> 1) ^ swv(key_v)) + 8 * (r & 1)) ^ (32u * db);
#pragma unroll
  for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(va[i]));
  asm volatile("" : "+v"(ka[0]), "+v"(ka[1]), "+v"(sa));

  // A step takes the softmax of its tile t between the products of two others: S of tile t + 1 (qk)
  // and the output of tile t - 1 (pv), so that no product waits for this tile's exponentials nor
  // they for it. The softmax is dealt over 8 slices of 2 elements; with them go qk n: key block
  // n / 2, q's hi part, then its lo part (two in each of the first 4 slices: their results are the
  // first that the next step needs), and pv n: key half n / 4, dim blocks 2 (n % 4) and the next.
  // (Products and softmax of one tile in turn: 4 windows of 32 over 2048 keys 22.9 us instead of
  // 20.5, 1 x 8192 tokens 349 instead of 330.)
  typedef __attribute__((address_space(3))) const u32x4_v* lds_u4_t;
  typedef __attribute__((address_space(3))) s16x4_v* tr_ptr_t;
  i32x8_v kf[2];
  s16x4_v vw[2][4][2];
  f32x4_v next[4];  // S of the next tile
  float s[16];      // S of this one: key 8 g + i, or 32 + 8 g + i - 8
  uint4 pn[2];      // P of this tile, and of the one before
  bf16x8_v pf[2];
  float m = NEG_BIG, l = 0.0f;  // (l: this lane's 16 keys of every tile)
  f32x4_v acc[8];
  float run_m = NEG_BIG, run_l = 0.0f;
  f32x4_v run_top = {0.0f, 0.0f, 0.0f, 0.0f};
  typedef __attribute__((address_space(3))) f32x4_v* park_t;
  const park_t parked = (park_t)(lds0 + kParkedAt + 16 * tid);  // vector i: + 64 NW i
  if constexpr (!FANOUT) {
#pragma unroll
    for (int i = 0; i < kParked; ++i) parked[64 * NW * i] = run_top;
  }
#pragma unroll
  for (int db = 0; db < 8; ++db) acc[db] = f32x4_v{0.0f, 0.0f, 0.0f, 0.0f};
  pf[0] = pf[1] = bf16x8_v{};
  auto read_k = [&](auto j_, auto buf) {
    constexpr int j = decltype(j_)::value;
    const uint32_t at = buf * kKTile + (32 * (j >> 1) + 4 * (j & 1)) * D;  // (swk is the same for all j)
    const u32x4_v k0 = *(lds_u4_t)(ka[0] + at);
    const u32x4_v k1 = *(lds_u4_t)(ka[1] + at);
    kf[j & 1] = i32x8_v{(int)k0.x, (int)k0.y, (int)k0.z, (int)k0.w,
                    (int)k1.x, (int)k1.y, (int)k1.z, (int)k1.w};
  };
  // V fragments: A = V^T rows 16 db + r (dims), columns 32 kb + 8 g .. +7 (keys), by two
  // transpose reads (extend_attention.hip). They go out in groups of 4, each before the products
  // of the one before it.
  auto read_v = [&](auto n_, auto buf) {  // group n: key half n / 2, dim blocks 4 (n % 2) .. +3
    constexpr int n = decltype(n_)::value;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = va[4 * (n & 1) + i] + buf * kTileBytes + 8192 * (n >> 1);
      vw[n & 1][i][0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)at);
      vw[n & 1][i][1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)(at + 1024));
    }
  };
  auto qk = [&](auto n_, int ks) {
    constexpr int n = decltype(n_)::value, j = n >> 1;
    constexpr bool lo = (n & 1) != 0;
    // (the scale operands' byte is an immediate: key block j of ks, hi or lo of the row's scale)
    if constexpr (lo)
      next[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kf[j & 1], qf.lo, next[j], 0, 0, j, ks, 1, qf.scale);
    else
      next[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
          kf[j & 1], qf.hi, f32x4_v{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, j, ks, 0, qf.scale);
  };
  auto pv = [&](auto n_) {
    constexpr int n = decltype(n_)::value;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int w = 2 * (n & 1) + i;
      const bf16x8_v vf = __builtin_bit_cast(
          bf16x8_v, static_cast<s16x8_v>(__builtin_shufflevector(
                        vw[(n >> 1) & 1][w][0], vw[(n >> 1) & 1][w][1], 0, 1, 2, 3, 4, 5, 6, 7)));
      f32x4_v& a = acc[2 * (n & 3) + i];
      a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n >> 2], a, 0, 0, 0);
    }
  };
  auto take_scores = [&] {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = next[i >> 2][i & 3];
  };
  auto each = [](auto f) {  // f(0) .. f(7), as constants
    f(std::integral_constant<int, 0>{}); f(std::integral_constant<int, 1>{});
    f(std::integral_constant<int, 2>{}); f(std::integral_constant<int, 3>{});
    f(std::integral_constant<int, 4>{}); f(std::integral_constant<int, 5>{});
    f(std::integral_constant<int, 6>{}); f(std::integral_constant<int, 7>{});
  };
  typedef std::integral_constant<int, 0> c0;
  typedef std::integral_constant<int, 1> c1;
  typedef std::integral_constant<int, 2> c2;
  typedef std::integral_constant<int, 3> c3;
  auto barrier = [&] {
    // Every load has landed (they had a whole tile's time) and every wave is done with the buffers
    // that are written next.
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  auto fold_split = [&](float om, float ol) {  // the state of a split that is complete
    const FoldScale f = fold_scale(run_m, om);
    run_l = fold_elem(run_l, pair32_sum(pair16_sum(ol)), f);
    run_m = f.mn;
#pragma unroll
    for (int db = 0; db < 8; ++db) {
      f32x4_v a = db < kParked ? parked[64 * NW * db] : run_top;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = fold_elem(a[i], acc[db][i], f);
      if (db < kParked) parked[64 * NW * db] = a;
      else run_top = a;
    }
  };

  // Tile t's step; buf: t & 1. MASK: some key of it may be hidden from some row. FIRST: of a split.
  auto step = [&](auto mask, auto first, int t, auto buf) {
    constexpr bool kMask = decltype(mask)::value, kFirst = decltype(first)::value;
    barrier();
    const bool mine = !kMask || t <= w_tiles;  // (at w_tiles the tile before is still to be added)
    int ks = 0;
    if (mine) {
      ks = *(__attribute__((address_space(3))) const int*)(sa + 64 * other(buf));
      read_v(c0{}, other(buf));
      read_k(c0{}, other(buf));
      read_k(c1{}, other(buf));
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < KP; ++i)  // (not converted ahead of the barrier)
      asm volatile("" : "+v"(raw[i]), "+v"(sc0.x[i]), "+v"(scales_in.x[i]));
    store_v(sc0, buf);
    store_scales(scales_in, buf);
    sc0 = sc1;
    sc1 = scales_in;
    load_v(sl1);
    check(sl3);
    scales_in = load_scales(sl3);
    const PerKey k_at = sl2;
    sl1 = sl2;
    sl2 = sl3;
    sl3 = load_slots(t + 4);
    __builtin_amdgcn_sched_barrier(0);
    if (t + 2 < t_end) load_k(k_at, buf);  // last: a wait for an earlier load would include the DMA
    __builtin_amdgcn_sched_barrier(0);
    if (!mine) return;
    const float om = m, ol = l;
    if constexpr (kFirst) {
      m = NEG_BIG;
      l = 0.0f;
    }
    bool vis[16];
    float tmax = NEG_BIG;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if constexpr (kMask) {
        vis[i] = (t * BN + 32 * (i >> 3) + 8 * g + (i & 7) <= q_abs) & row_ok;
        tmax = fmaxf(tmax, vis[i] ? s[i] : NEG_BIG);
      } else {
        tmax = fmaxf(tmax, s[i]);
      }
    }
    // Each lane looks at its own 16 scores: only where one of them is LAZY_T above its row's
    // reference maximum (seldom, but for a split's first tile) is the row's maximum taken.
    const bool moved = kFirst || __builtin_amdgcn_ballot_w64(tmax * sc2 > m + LAZY_T) != 0;
    float rescale = 1.0f;
    if (moved) {
      const float mc = pair32_max(pair16_max(tmax)) * sc2;
      const float m_used = mc > m + LAZY_T ? mc : m;
      rescale = exp2_fast(m - m_used);
      m = m_used;
      if constexpr (!kFirst) l *= rescale;
    }
    // (A wave with products to issue goes first: of two waves on a SIMD one is ahead, and its products
    // run beside the other's conversions and loads. 5 ragged chunks 108 -> 101 us, 1 x 8192 tokens
    // 330 -> 323.)
    __builtin_amdgcn_s_setprio(1);
    each([&](auto n_) {
      constexpr int n = decltype(n_)::value;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (n < 4) qk(std::integral_constant<int, 2 * (n & 3)>{}, ks);
      if constexpr (n == 0) read_v(c1{}, other(buf));
      if constexpr (n == 1) read_k(c2{}, other(buf));
      if constexpr (n == 2) read_k(c3{}, other(buf));
      if constexpr (n == 2) read_v(c2{}, other(buf));
      if constexpr (n == 4) read_v(c3{}, other(buf));
      float p[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        p[i] = exp2_fast(__builtin_fmaf(s[2 * n + i], sc2, -m));
        if constexpr (kMask) p[i] = vis[2 * n + i] ? p[i] : 0.0f;
        l += p[i];
      }
      reinterpret_cast<uint32_t*>(&pn[n >> 2])[n & 3] = pack_bf16x2(p[0], p[1]);
      pv(n_);
      if constexpr (n < 4) qk(std::integral_constant<int, 2 * (n & 3) + 1>{}, ks);
    });
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    // (here, not where the next step uses them: past the branches below they would move there)
    asm volatile("" : "+v"(next[0]), "+v"(next[1]), "+v"(next[2]), "+v"(next[3]));
    asm volatile("" : "+v"(l), "+v"(pn[0].x), "+v"(pn[0].y), "+v"(pn[0].z), "+v"(pn[0].w),
                 "+v"(pn[1].x), "+v"(pn[1].y), "+v"(pn[1].z), "+v"(pn[1].w));
    if constexpr (kFirst) {
      // (before the first split: nothing, times what lay in the LDS)
      if (!FANOUT && t > t_begin) fold_split(om, ol);
#pragma unroll
      for (int db = 0; db < 8; ++db) acc[db] = f32x4_v{0.0f, 0.0f, 0.0f, 0.0f};
    } else if (moved) {  // (x * 1 == x for the rows that did not)
#pragma unroll
      for (int db = 0; db < 8; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[db][i] *= rescale;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) pf[i] = __builtin_bit_cast(bf16x8_v, pn[i]);
    take_scores();
  };

  // S of the first tile.
  barrier();
  {
    const int ks = *(__attribute__((address_space(3))) const int*)sa;
    read_k(c0{}, c0{});
    each([&](auto n_) {
      constexpr int n = decltype(n_)::value;
      if constexpr (n < 6 && n % 2 == 0) read_k(std::integral_constant<int, n / 2 + 1>{}, c0{});
      qk(n_, ks);
    });
    take_scores();
  }
  // Tiles that every row of the workgroup sees whole, in pairs (their buffers' addresses are
  // immediates), then the others with the mask: one loop each, split by split (a branch between
  // the kinds in one loop, or the fold in it, costs a copy of the accumulators each turn).
  const int t_full = (prefix + mtile * ROWS + 1) / BN;
  constexpr std::true_type yes;
  constexpr std::false_type no;
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
      if constexpr (n == 0) read_v(c1{}, buf);
      if constexpr (n == 2) read_v(c2{}, buf);
      if constexpr (n == 4) read_v(c3{}, buf);
      __builtin_amdgcn_sched_barrier(0);
      pv(n_);
    });
  }
  if constexpr (FANOUT) {
    l = pair32_sum(pair16_sum(l));
    if (!row_ok) return;
    const int64_t pr = split * items + prow;
#pragma unroll
    for (int db = 0; db < 8; ++db)
      *reinterpret_cast<f32x4_v*>(part_a + pr * D + 16 * db + 4 * g) = acc[db];
    if (g == 0) {
      part_ml[2 * pr] = m;
      part_ml[2 * pr + 1] = l;
      if (split == 0) part_n[prow] = nsplits;
    }
  } else {
    fold_split(m, l);
    RowState run{run_m, run_l, {}};
#pragma unroll
    for (int db = 0; db < 8; ++db) run.acc[db] = db < kParked ? parked[64 * NW * db] : run_top;
    if (row_ok) store_row(o + prow * D, run, g);
  }
}

// Whether a grid of fewer than 512 workgroups fans out. Walking its keys in one workgroup takes about
// 6 + 1.1 us a tile; fanned out, the launches take 18 us and the saved states of total_q rows in
// every split 8.5 us a thousand. Walked and fanned out, us: 1 x 512 tokens 14 and 23, 1 x 1024 23 and
// 38, 2 x 500 over 2000 48 and 66, 4 x 200 over 1000 27 and 35, 1 x 700 over 4000 76 and 78, 16 x 32
// over 2048 40 and 35, 8 x 64 over 3000 53 and 40, 4 x 32 over 2048 39 and 20, 1 x 256 over 8000 126
// and 55.
bool fans_out(int batch, int64_t total_q, int num_kv_heads, int max_extend_len, int max_kv_len) {
  const int64_t groups = static_cast<int64_t>(batch) * num_kv_heads * ceil_div(max_extend_len, BQ);
  const int64_t states = total_q * ceil_div(max_kv_len, kSplit);
  return groups < 512 && 110 * static_cast<int64_t>(ceil_div(max_kv_len, BN)) > 1200 + states * 85 / 100;
}

}  // namespace
}  // namespace sid

using namespace sid;

extern "C" int64_t sid_extend_attention_fp8_workspace_bytes(int batch, int64_t total_q,
                                                            int num_q_heads, int num_kv_heads,
                                                            int max_extend_len, int max_kv_len) {
  if (batch <= 0 || total_q <= 0 || max_extend_len <= 0 || max_kv_len <= 0) return 0;
  if (!fans_out(batch, total_q, num_kv_heads, max_extend_len, max_kv_len)) return 0;
  // per (split, row, head): 128 accumulator floats + (m, l); per (row, head): split count
  const int64_t splits = ceil_div(max_kv_len, kSplit);
  return (splits * (D + 2) + 1) * total_q * num_q_heads * static_cast<int64_t>(sizeof(float));
}

extern "C" int sid_extend_attention_fp8_fwd(
    const void* q, const void* k_cache, const void* v_cache, const void* kv_scales,
    const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices, int batch,
    int64_t total_q, int num_q_heads, int num_kv_heads, int head_dim, int64_t num_slots,
    int max_extend_len, int max_kv_len, float sm_scale, void* workspace, int64_t workspace_bytes,
    void* o, void* stream) {
  const char* name = "extend_attention_fp8";
  const ExtendPlan p = extend_plan(name, q, k_cache, v_cache, qo_indptr, kv_indptr, kv_indices, o,
                                   batch, total_q, num_q_heads, num_kv_heads, head_dim, num_slots,
                                   max_extend_len, max_kv_len, kSplit,
                                   sid_extend_attention_fp8_workspace_bytes(
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
  auto launch = [&](auto kern, int nw, dim3 grid, int mtiles, int across) {
    hipLaunchKernelGGL(kern, grid, dim3(nw * 64), 0, s, (const bf16_t*)q,
                       (const uint8_t*)k_cache, (const uint8_t*)v_cache,
                       (const uint16_t*)kv_scales, qo_indptr, kv_indptr, kv_indices, batch,
                       num_q_heads, num_kv_heads, num_slots, sm_scale, mtiles, per_round, ordered,
                       across, p.items, (bf16_t*)o, p.part_a, p.part_ml, p.part_n);
    return check_launch(name);
  };
  if (p.fanout) {
    const int rc = launch(extend_fp8_kernel<4, true>, 4,
                          dim3(batch, num_kv_heads, p.mtiles * p.splits), p.mtiles, 0);
    return rc != SID_OK ? rc : extend_merge(name, p, qo_indptr, batch, num_q_heads, o, s);
  }
  const int mtiles = ceil_div(max_extend_len, p.rows);
  const int64_t places = static_cast<int64_t>(batch) * mtiles;
  const int across = static_cast<int>(std::min<int64_t>(places, kMaxGridX / num_kv_heads));
  const int64_t down = (places + across - 1) / across;
  SID_REQUIRE(places < (1ll << 30) && down <= 65535, "%s: grid too large", name);
  const dim3 grid(static_cast<unsigned>(across) * num_kv_heads, static_cast<unsigned>(down));
  return p.rows == 64 ? launch(extend_fp8_kernel<8, false>, 8, grid, mtiles, across)
                      : launch(extend_fp8_kernel<4, false>, 4, grid, mtiles, across);
}
