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
//
// Workgroups are of 4 waves and 32 query positions, two to a CU, as an independent workgroup fills the
// waits of the other best: 8 waves of 64 positions, and 4 waves with two row sets that share each fragment,
// took 3 to 40 % longer. Over 8 kv heads of 2 query heads, us by the card: 1 x 8192 296-330 (930-833
// TFLOP/s; the 8-bit pool's kernel 349 beside 336), 4 x 2048 93-101, 1 x 2048 30-33, 4 x 32 at 2048 keys 17-19.
// Of 4 x 2048 the vector ALU (softmax, V to bf16) issues for 56 % and the matrix units and the LDS (each wave reads all of V for its 16 rows) are
// busy for 33 % and 44 %, in each other's shadow: what bounds it is each wave's own chain, two a SIMD. 16 x 512 to 1 x 8192
// (8192 queries each) take 6.7 us a workgroup, its first loads, first S and last fold, and 1.05 us a tile of 64 keys
// beside it, within 5 %: 27 of 4 x 2048's 96 us, as a CU's places take four workgroups one after the other. A third
// workgroup a CU has no room: the walking form is compiled to 256 registers, and its LDS is 74752 bytes, 33280
// of them the parked rows.
#include "extend_codes.h"
#include "kv_fp4.h"

#include <algorithm>

namespace sid {
namespace {

constexpr int NW = 4;  // waves of a workgroup
// Keys per split: the unit in which a row's state is folded. (With 1024 a prompt of 8192 takes 5 % less,
// but 4 x 32 queries at 2048 keys, which fan out by splits, 20.7 us instead of 17.)
constexpr int kSplit = 512;
constexpr int kSplitTiles = kSplit / BN;
// How far above its row's reference maximum a score may be: 24 octaves, as p. (A split's sums of p v are
// then at most 2^33 of its largest |v|: finite below 2^94.)
constexpr float kLazySum = 16777216.0f;

// ---- LDS ---------------------------------------------------------------------------------
//
// Two tiles of 64 keys, as four sub-tiles of 32. K stays in codes, 64 bytes a key: 16-byte unit u of a
// key's row holds block u ^ swk(key), which spreads a fragment's 16 rows over the banks. V
// is bf16 (swv). Beside them K's scale bytes as the matrix instruction takes them: half-word l of a
// sub-tile holds lane l's for its two key blocks.
constexpr int BS = 32;  // keys of a sub-tile
constexpr int kKSub = BS * D / 2, kVSub = BS * D * 2, kScaleSub = 128;
constexpr int kVAt = 4 * kKSub;
constexpr int kScalesAt = kVAt + 4 * kVSub;
// The rows' folded state stays in the LDS between two folds, 512 keys apart (the registers hold the
// state of the split in work): a lane's 8 accumulator vectors, and the rows' m and l.
constexpr int kRunAt = kScalesAt + 4 * kScaleSub;
constexpr int lds_bytes(bool fanout) { return kRunAt + (fanout ? 0 : NW * (8 * 1024 + 128)); }

// 0, 2, 3, 1 for the four groups of rows: a read of 16 bytes takes lanes 0-3, 12-15, 20-27 and their like at
// once, whose blocks are then four different ones. (0, 1, 2, 3: 6.9 M cycles of conflicts in 4 x 2048, and
// 1 % longer. 4.6 M are left, of V's writes: half of the lanes writing their words in another order ends
// them, but its selects cost what that gains.)
__device__ __forceinline__ int swk(int key) {
  const int x = (key >> 3) & 3;
  return ((x << 1) & 3) ^ 3 * (x >> 1);
}

// Workgroup = (request, kv head, 8 NW query positions), NW waves; wave w: 16 positions of query head
// w / (NW / 2). FANOUT: the workgroup computes one split and saves its state for the fold; else it
// walks the splits in order.
template <bool FANOUT>
__global__ void __launch_bounds__(NW * 64, 2) extend_fp4_kernel(
    const bf16_t* __restrict__ q, const uint8_t* __restrict__ k_cache,
    const uint8_t* __restrict__ v_cache, const uint2* __restrict__ kv_scales,
    const int32_t* __restrict__ qo_indptr, const int32_t* __restrict__ kv_indptr,
    const int32_t* __restrict__ kv_indices, int batch, int num_q_heads, int num_kv_heads,
    int64_t num_slots, float sm_scale, int mtiles, int per_round, int ordered, int across,
    int64_t items, bf16_t* __restrict__ o, float* __restrict__ part_a,
    float* __restrict__ part_ml, int32_t* __restrict__ part_n) {
  __shared__ __align__(1024) char lds[lds_bytes(FANOUT)];
  constexpr int ROWS = 8 * NW;
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

  // ---- staging. A step works on a tile of 64 keys, as two sub-tiles 2 t and 2 t + 1, and stages K of
  // tile t + 2 and V of t + 1. A thread's piece is 32 codes: key t / 4 of a tile, block t % 4. K's go to
  // the LDS by DMA during the step; V's through registers, where they become bf16 with their scale (once
  // for all waves) at the step's end, when those of t + 2 go out. No branch that differs between steps
  // guards a load with a register result (past the sequence's end its last key is read again): such a
  // load is waited for where the branch ends.
  const int32_t* idx = kv_indices + kv_start;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char_t)lds));
  const uint32_t max_slots = static_cast<uint32_t>(min<int64_t>(num_slots, 0x7fffffff));
  const int my_key = tid >> 2, my_blk = tid & 3;
  auto load_slot = [&](int tile) -> uint32_t { return idx[min(tile * BN + my_key, kv_len - 1)]; };
  // Out of range: slot 0. (Looked at where a slot is used first: at its load, it would be waited
  // for.)
  auto checked = [&](uint32_t slot) { return slot < max_slots ? slot : 0u; };
  const uint32_t row_bytes = static_cast<uint32_t>(num_kv_heads) * (D / 2);
  // Of the row in a pool of codes; the scales' are an eighth of it.
  auto offset = [&](uint32_t slot) { return static_cast<uint64_t>(slot) * row_bytes; };
  const uint8_t* ksrc = k_cache + h_kv * (D / 2) + 16 * (my_blk ^ swk(my_key));
  const uint8_t* vsrc = v_cache + h_kv * (D / 2) + 16 * my_blk;
  const uint8_t* sbase = reinterpret_cast<const uint8_t*>(kv_scales + h_kv);
  auto load_k = [&](uint64_t off, int buf) { dma16(ksrc + off, lds0 + 2 * buf * kKSub + 1024u * wave); };
  auto load_v = [&](uint64_t off) { return *reinterpret_cast<const u32x4_v*>(vsrc + off); };
  auto load_scales = [&](uint64_t off) { return *reinterpret_cast<const uint2*>(sbase + (off >> 3)); };
  // A NaN vector must reach the queries that see its key and no others, but a hidden key's value is
  // multiplied by p = 0, which leaves a NaN. So a key whose V is NaN gets a NaN scale for K (E8M0's
  // 255: NaN scores, and a hidden key's scores are never used) and values of next to nothing (scale
  // byte 0).
  const uint32_t sdst = kScalesAt + (my_key >> 5) * kScaleSub +
                        2 * (16 * my_blk + 4 * ((my_key >> 3) & 3) + (my_key & 3)) + ((my_key >> 2) & 1);
  auto store_scales = [&](uint2 sc, int buf) {
    const uint32_t k = sc.x >> (8 * my_blk), v = (sc.y >> (8 * my_blk)) & 255u;
    reinterpret_cast<uint8_t*>(lds)[sdst + 2 * buf * kScaleSub] = static_cast<uint8_t>(v == kFp4ScaleNaN ? v : k);
  };
  const uint32_t vdst = lds0 + kVAt + 256 * my_key + 16 * ((4 * my_blk) ^ swv(my_key));
  auto store_v = [&](const u32x4_v& codes, uint32_t scales, int buf) {
    const uint32_t byte = (scales >> (8 * my_blk)) & 255u;
    const float s = fp4_scale(byte == kFp4ScaleNaN ? 0u : byte);
    typedef __attribute__((address_space(3))) u32x4_v* lds_w_t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 x = fp4_to_bf16x8(codes[i], s);
      *(lds_w_t)((vdst ^ (16u * i)) + 2 * buf * kVSub) = u32x4_v{x.x, x.y, x.z, x.w};
    }
  };

  // The first loads, in the order of their latencies: slots and q, then what the slots name; q is
  // split while those are under way. (t_begin is a split's first tile: even.)
  const uint32_t slot0 = load_slot(t_begin), slot1 = load_slot(t_begin + 1);
  uint32_t next_slot = load_slot(t_begin + 2);
  const QRaw q_raw = load_q(q + prow * D, g);
  __builtin_amdgcn_sched_barrier(0);
  const uint64_t off0 = offset(checked(slot0)), off1 = offset(checked(slot1));
  const uint2 s0 = load_scales(off0), s1 = load_scales(off1);
  const u32x4_v raw0 = load_v(off0);
  u32x4_v raw = load_v(off1);
  __builtin_amdgcn_sched_barrier(0);
  load_k(off0, 0);
  load_k(off1, 1);
  __builtin_amdgcn_sched_barrier(0);
  const QRow qf = split_q(q_raw, row_ok);
  __builtin_amdgcn_sched_barrier(0);
  store_scales(s0, 0);
  store_scales(s1, 1);
  store_v(raw0, s0.y, 0);
  uint32_t v_scales = s1.y;
  __builtin_amdgcn_sched_barrier(0);

  // LDS addresses of a lane's fragments in sub-tile 0, kept in registers.
  // S^T = K Q^T: row m of a sub-tile's key block j is key 8 (m / 4) + 4 j + m % 4, so a lane ends with
  // the scores of keys 8 g .. +7 of its queries.
  const int key_a0 = 8 * (r >> 2) + (r & 3);
  uint32_t ka = lds0 + key_a0 * (D / 2) + 16 * (g ^ swk(key_a0)), sa = lds0 + kScalesAt + 2 * lane;
  const int key_v = 8 * g + (r >> 2);
  uint32_t va[8];
#pragma unroll
  for (int db = 0; db < 8; ++db) {
    va[db] = (lds0 + kVAt + key_v * 256 + 16 * (((r & 3) >> 1) ^ swv(key_v)) + 8 * (r & 1)) ^ (32u * db);
    asm volatile("" : "+v"(va[db]));
  }
  asm volatile("" : "+v"(ka), "+v"(sa));

  // Sub-tile u takes its softmax between the products of two others: S of u + 1 (qk) and the output
  // of u - 1 (pv), so that no product waits for its exponentials nor they for it. The softmax is dealt
  // over 4 slices of 2 elements a row set; with slice n go qk n: key block n / 2, q's hi part, then its
  // lo part, and pv n + 1: dim blocks 2 n + 2 and the next (pv 0 with the maxima before them). The
  // fragments are in registers when a sub-tile begins: they are read during the one before, each as
  // soon as its predecessor is used up, so that neither a barrier nor the LDS is waited for.
  typedef __attribute__((address_space(3))) const u32x4_v* lds_u4_t;
  typedef __attribute__((address_space(3))) s16x4_v* tr_ptr_t;
  u32x4_v kf[2];
  int ks;  // kf's scales
  s16x8_v vw[4][2];
  f32x4_v s[2][2];  // [u % 2]: S of this sub-tile and of the next
  uint4 p4[2];      // [u % 2]: P of this sub-tile and of the one before
  float m = NEG_BIG, l = 0.0f;  // (l: this lane's 8 keys of every sub-tile)
  f32x4_v acc[8];
  typedef __attribute__((address_space(3))) f32x4_v* park_t;
  const park_t parked = (park_t)(lds0 + kRunAt + 16 * tid);  // vector db: + 64 NW db
  typedef __attribute__((address_space(3))) f32x2_fp4* row_t;
  const row_t run_ml = (row_t)(lds0 + kRunAt + NW * 8 * 1024 + 8 * (16 * wave + r));  // the row's m and l
  constexpr f32x4_v zero4 = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int db = 0; db < 8; ++db) {
    acc[db] = zero4;
    if constexpr (!FANOUT) parked[64 * NW * db] = zero4;
  }
  if constexpr (!FANOUT) *run_ml = f32x2_fp4{NEG_BIG, 0.0f};
  p4[0] = p4[1] = make_uint4(0, 0, 0, 0);
  auto read_k = [&](int at) {
    ks = *(__attribute__((address_space(3))) const uint16_t*)(sa + at * kScaleSub);
#pragma unroll
    for (int j = 0; j < 2; ++j) kf[j] = *(lds_u4_t)(ka + at * kKSub + 4 * j * (D / 2));
  };
  // V fragments: A = V^T rows 16 db + r (dims), columns 8 g .. +7 (keys), by two transpose reads
  // (extend_attention.hip): those of pv n.
  auto read_v = [&](int n, int at) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t a = va[2 * n + i] + at * kVSub;
      vw[n][i] = __builtin_shufflevector(__builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)a),
                                         __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)(a + 1024)), 0,
                                         1, 2, 3, 4, 5, 6, 7);
    }
  };
  auto qk = [&](auto n_, f32x4_v (&to)[2]) {
    constexpr int n = decltype(n_)::value, j = n >> 1;
    const u32x4_v kk = kf[j];
    const i32x8_v a{(int)kk.x, (int)kk.y, (int)kk.z, (int)kk.w, 0, 0, 0, 0};
    // (formats 4 and 0: e2m1 and e4m3; the scale operands' byte is an immediate: key block j of ks,
    // hi or lo of the row's scale)
    if constexpr ((n & 1) != 0)
      to[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, qf.lo, to[j], 4, 0, j, ks, 1, qf.scale);
    else
      to[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, qf.hi, zero4, 4, 0, j, ks, 0, qf.scale);
  };
  // FRESH: acc holds nothing of this split yet.
  auto pv = [&](auto fresh, int n, int i, const uint4& p) {
    f32x4_v& a = acc[2 * n + i];
    a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_v, vw[n][i]),
                                                __builtin_bit_cast(bf16x8_v, p),
                                                decltype(fresh)::value ? zero4 : a, 0, 0, 0);
  };
  auto each = [](auto f) {  // f(0) .. f(3), as constants
    f(std::integral_constant<int, 0>{}); f(std::integral_constant<int, 1>{});
    f(std::integral_constant<int, 2>{}); f(std::integral_constant<int, 3>{});
  };
  typedef std::integral_constant<int, 0> c0;
  typedef std::integral_constant<int, 1> c1;
  constexpr std::true_type yes;
  constexpr std::false_type no;
  auto point = [] { __builtin_amdgcn_sched_barrier(0); };
  // The state (om, ol) and acc of a split that is complete, into the row's.
  auto fold_split = [&](float om, float ol) {
    const f32x2_fp4 ml = *run_ml;
    const FoldScale f = fold_scale(ml.x, om);
    *run_ml = f32x2_fp4{f.mn, fold_elem(ml.y, pair32_sum(pair16_sum(ol)), f)};  // (4 lanes, the same bits)
#pragma unroll
    for (int db = 0; db < 8; ++db) {
      f32x4_v a = parked[64 * NW * db];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = fold_elem(a[i], acc[db][i], f);
      parked[64 * NW * db] = a;
    }
  };

  // Half h of tile t: sub-tile u = 2 t + h. MASK: some key of it may be hidden from some row. FIRST: of a
  // split (it finishes the one before). FRESH: the second of a split.
  auto half = [&](auto mask, auto first, auto fresh, auto h_, int t, auto buf, auto tail) {
    constexpr bool kMask = decltype(mask)::value, kFirst = decltype(first)::value;
    constexpr int h = decltype(h_)::value;
    const int v_at = 2 * buf + h, k_at = 2 * other(buf) + h;  // what is read here: V of u, K of u + 2
    const f32x4_v (&sc)[2] = s[h];
    bool vis[8];
    if constexpr (kMask) {
#pragma unroll
      for (int i = 0; i < 8; ++i) vis[i] = (t * BN + BS * h + 8 * g + i <= q_abs) & row_ok;
    }
    auto seen = [&](int i) { return !kMask || vis[i] ? sc[i >> 2][i & 3] : NEG_BIG; };
    point();
    __builtin_amdgcn_s_setprio(1);
    pv(fresh, 0, 0, p4[1 - h]);
    pv(fresh, 0, 1, p4[1 - h]);
    point();
    const float om = m, ol = l;
    auto row_max = [&] {
      float tmax = NEG_BIG;
#pragma unroll
      for (int i = 0; i < 8; ++i) tmax = fmaxf(tmax, seen(i));
      return pair32_max(pair16_max(tmax)) * sc2;
    };
    if constexpr (kFirst) {
      m = row_max();
      l = 0.0f;
    }
    // (While a product runs, a wave can issue only what follows it in program order, and a second
    // product behind it waits for the first. So between two products stands about as much of the
    // softmax as the first one takes: 34 cycles a qk, 16 a pv. The priority lets the other workgroup's wave
    // of the SIMD stage while this one keeps the matrix unit fed: 1.5 % of 1 x 8192.)
    each([&](auto n_) {
      constexpr int n = decltype(n_)::value, j = n >> 1, i0 = 2 * (n & 1);
      float x[2], p[2];
      point();
      read_v(n, v_at);
#pragma unroll
      for (int i = 0; i < 2; ++i) x[i] = __builtin_fmaf(sc[j][i0 + i], sc2, -m);
      point();
      qk(n_, s[1 - h]);
      point();
      p[0] = exp2_fast(x[0]);
      p[1] = exp2_fast(x[1]);
      point();
      if constexpr (n == 3) read_k(k_at);
      if constexpr (n < 3) pv(fresh, n + 1, 0, p4[1 - h]);
      point();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (kMask) p[i] = vis[2 * n + i] ? p[i] : 0.0f;
        l += p[i];
      }
      reinterpret_cast<uint32_t*>(&p4[h])[n] = pack_bf16x2(p[0], p[1]);
      point();
      if constexpr (n < 3) pv(fresh, n + 1, 1, p4[1 - h]);
      point();
    });
    // (here, not where they are used: past the branches below they would move there)
    asm volatile("" : "+v"(s[1 - h][0]), "+v"(s[1 - h][1]));
    asm volatile("" : "+v"(l), "+v"(p4[h].x), "+v"(p4[h].y), "+v"(p4[h].z), "+v"(p4[h].w));
    __builtin_amdgcn_s_setprio(0);
    tail();
    if constexpr (kFirst) {
      if (!FANOUT && t > t_begin) fold_split(om, ol);
    } else {
      // A row's reference maximum is that of its split's first sub-tile until one of its scores is 24
      // octaves above it: P's precision does not depend on its size. Such a score makes its lane's sum grow by
      // more than kLazySum (at the border the roundings decide); only where one does (hardly ever) are the
      // rows' maxima taken, their state brought to them and P worked out again. Each row goes by the sums
      // of its own four lanes there, so whether it moves does not depend on who shares its wave. That is
      // looked at here, after the products, as nothing before has to wait for it. (By the sums, not by the
      // scores' maximum: 5 operations fewer of some 50, 2 % of 1 x 8192.)
      uint64_t up = __builtin_amdgcn_ballot_w64(l - ol > kLazySum);
      if (__builtin_expect(up != 0, false)) {
        up |= up >> 32 | up << 32;  // a row's four lanes are 16 apart
        up |= up >> 16 | up << 48;
        const float mc = row_max();  // (of a row that moves some 20 octaves above m, or more)
        const float m_used = __builtin_amdgcn_inverse_ballot_w64(up) ? mc : m;
        const float rescale = exp2_fast(m - m_used);  // (x * 1 == x for the rows that stay)
        m = m_used;
        l = ol * rescale;
        uint4 w;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          float p[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            p[i] = exp2_fast(__builtin_fmaf(sc[n >> 1][2 * (n & 1) + i], sc2, -m));
            if constexpr (kMask) p[i] = vis[2 * n + i] ? p[i] : 0.0f;
            l += p[i];
          }
          reinterpret_cast<uint32_t*>(&w)[n] = pack_bf16x2(p[0], p[1]);
        }
        p4[h] = w;
        // (Out of a product with zeros: vectors whose elements change in a branch would be copied, all of
        // them, on the way past it.)
#pragma unroll
        for (int db = 0; db < 8; ++db) {
          const f32x4_v a = acc[db];
          acc[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              bf16x8_v{}, bf16x8_v{}, f32x4_v{a[0] * rescale, a[1] * rescale, a[2] * rescale, a[3] * rescale},
              0, 0, 0);
        }
      }
    }
  };

  auto step = [&](auto mask, auto first, int t, auto buf) {
    constexpr bool kMask = decltype(mask)::value;
    // Every wave is done with the tiles that are written over next, and K has landed (it had a whole
    // tile's time). V is still under way, the last load that went out.
    point();
    asm volatile("s_waitcnt vmcnt(1) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    point();
    const uint64_t off = offset(checked(next_slot));  // of tile t + 2
    const uint2 scales = load_scales(off);
    next_slot = load_slot(t + 3);
    point();
    load_k(off, buf);  // last: a wait for an earlier load would include the DMA
    point();
    auto stage = [&] {  // at the step's end
      store_v(raw, v_scales, other(buf));
      point();
      raw = load_v(off);
      v_scales = scales.y;
      point();
      store_scales(scales, buf);
      point();
    };
    if (!kMask || t <= w_tiles) {  // (at w_tiles the sub-tile before is still to be added)
      half(mask, first, no, c0{}, t, buf, [] {});
      half(mask, no, first, c1{}, t, buf, stage);
    } else {
      stage();
    }
  };

  // S of the first sub-tile.
  auto barrier = [&] {
    point();
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    point();
  };
  barrier();
  read_k(0);
#pragma unroll
  for (int n = 0; n < 4; ++n) vw[n][0] = vw[n][1] = s16x8_v{};
  each([&](auto n_) { qk(n_, s[0]); });
  read_k(1);
  // Tiles that every row of the workgroup sees whole, in pairs (their places in the rings are
  // immediates), then the others with the mask: one loop each, split by split (a branch between
  // the kinds in one loop, or the fold in it, costs a copy of the accumulators each turn).
  const int t_full = (prefix + mtile * ROWS + 1) / BN;
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
  // The last sub-tile's output. (A wave that left out the last tiles has P = 0 and finite values.)
  each([&](auto n_) {
    constexpr int n = decltype(n_)::value;
    pv(no, n, 0, p4[1]);
    pv(no, n, 1, p4[1]);
  });
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
    const f32x2_fp4 ml = *run_ml;
    RowState run{ml.x, ml.y, {}};
#pragma unroll
    for (int db = 0; db < 8; ++db) run.acc[db] = parked[64 * NW * db];
    if (row_ok) store_row(o + prow * D, run, g);
  }
}

// Whether a grid of fewer than 512 workgroups fans out: where walking its keys in one workgroup (about
// a microsecond a tile) takes longer than the launches (10) and the saved states of total_q rows in every
// split. Walked and fanned out, us: 1 x 32 queries at 700 keys 15.8 and 14.0, 4 x 32 at 2048 32 and 18, 1 x 64 at
// 16384 227 and 34, 16 x 32 at 2048 38 and 34; 1 x 512 12 and 21, 1 x 700 at 4000 63 and 70 (the line's
// wrong side, as 1 x 512 at 2048, 37 and 41), 16 x 32 at 1024 24 and 26, 32 x 32 at 2048 41 and 59,
// 64 x 8 at 1024 35 and 44.
bool fans_out(int batch, int64_t total_q, int num_kv_heads, int max_extend_len, int max_kv_len) {
  const int64_t groups = static_cast<int64_t>(batch) * num_kv_heads * ceil_div(max_extend_len, BQ);
  const int64_t states = total_q * ceil_div(max_kv_len, kSplit);
  return groups < 512 && 105 * static_cast<int64_t>(ceil_div(max_kv_len, BN)) > 1000 + states * 95 / 100;
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
  SID_REQUIRE(sm_scale >= 0.0f && sm_scale < INFINITY,
              "%s: sm_scale must be finite and not negative (the scores' maxima are taken before it)", name);
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
  const int per_round = max(1, cu_count() / num_kv_heads);
  auto launch = [&](auto kern, dim3 grid, int mtiles, int across) {
    hipLaunchKernelGGL(kern, grid, dim3(NW * 64), 0, s, (const bf16_t*)q, (const uint8_t*)k_cache,
                       (const uint8_t*)v_cache, (const uint2*)kv_scales, qo_indptr, kv_indptr,
                       kv_indices, batch, num_q_heads, num_kv_heads, num_slots, sm_scale, mtiles,
                       per_round, ordered, across, p.items, (bf16_t*)o, p.part_a, p.part_ml, p.part_n);
    return check_launch(name);
  };
  if (p.fanout) {
    const int rc = launch(extend_fp4_kernel<true>, dim3(batch, num_kv_heads, p.mtiles * p.splits),
                          p.mtiles, 0);
    return rc != SID_OK ? rc : extend_merge(name, p, qo_indptr, batch, num_q_heads, o, s);
  }
  const int mtiles = ceil_div(max_extend_len, 8 * NW);
  const int64_t places = static_cast<int64_t>(batch) * mtiles;
  const int across = static_cast<int>(std::min<int64_t>(places, kMaxGridX / num_kv_heads));
  const int64_t down = (places + across - 1) / across;
  SID_REQUIRE(places < (1ll << 30) && down <= 65535, "%s: grid too large", name);
  const dim3 grid(static_cast<unsigned>(across) * num_kv_heads, static_cast<unsigned>(down));
  return launch(extend_fp4_kernel<false>, grid, mtiles, across);
}
