// Rotary positions from frequencies, without a table: any even part of a head, pairs of halves or
// of neighbours, and the frequencies and gain of a context scaled beyond its trained length.
//
// The pair i of a head turns by gain (cos, sin)(2 pi pos f_i): f_i, in turns a position, comes as
// a 64-bit fraction of a turn, so pos f_i modulo a turn is the low 64 bits of an integer product.
// That is exact but for f_i's own 2^-65: off by pos 2^-62 radians, whatever the position, where a
// product in 32 bits is off by pos 2^-25 of its angle. What is left of it after whole quarter turns, at most
// an eighth of one either way, goes to fp32 with all its 62 bits (so a small angle's sine is as near, in
// proportion, as a large one's), and its sine and cosine to their Taylor sums (terms to x^9 and x^8: the
// first left out is 2e-9 and 2.5e-8). q and k are rounded once, to bf16.
//
// Bound: q and k read and written. A workgroup takes one token and works its rotary / 2 angles out once for
// all heads, into the LDS. (Two or four tokens a workgroup, in turn on one card: 64 tokens 2.7 us with one, 3.2 and 3.7; 8192 of
// 24 heads of 128 16.5, 16.9 and 17.3; with half of a head turned 18.1, 17.5 and 18.1, and 32768 of those 85, 78
// and 78, the one case that gains.) 8192 tokens in 16.5 us move 100 MB at 6.1 TB/s, half of it out of the
// last level cache.
#include "rowmath.h"

namespace sid {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 512;  // of a head: 4 KiB of the LDS

// (sin, cos) of a 64-bit fraction of a turn.
__device__ __forceinline__ float2 sincos_turns(uint64_t turns) {
  const uint32_t quarter = (static_cast<uint32_t>(turns >> 32) + 0x20000000u) >> 30;
  const int64_t rest = static_cast<int64_t>(turns - (static_cast<uint64_t>(quarter) << 62));
  const float x = static_cast<float>(rest) * 3.406121580086e-19f;  // 2 pi 2^-64 radians a unit
  const float y = x * x;
  const float s = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 362880.0f, -1.0f / 5040.0f), 1.0f / 120.0f),
                                   -1.0f / 6.0f), x);
  const float c = fmaf(y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 40320.0f, -1.0f / 720.0f), 1.0f / 24.0f), -0.5f),
                       1.0f);
  const float a = (quarter & 1) ? c : s, b = (quarter & 1) ? s : c;
  return make_float2((quarter & 2) ? -a : a, ((quarter + 1) & 2) ? -b : b);
}

struct RopeArgs {
  const bf16_t* q;
  const bf16_t* k;
  bf16_t* q_out;
  bf16_t* k_out;
  int64_t ldq, ldk, ldqo, ldko;  // elements between tokens
  const int64_t* positions;
  const uint64_t* turns;
  int64_t max_positions;
  float gain;
  int rotary, head_dim, q_heads, heads;  // heads: of q and k
};

// Where element 0 of a token's head lies, and where it goes.
__device__ __forceinline__ void head_at(const RopeArgs& a, int64_t t, int h, const bf16_t*& src,
                                        bf16_t*& dst) {
  if (h < a.q_heads) {
    src = a.q + t * a.ldq + static_cast<int64_t>(h) * a.head_dim;
    dst = a.q_out + t * a.ldqo + static_cast<int64_t>(h) * a.head_dim;
  } else {
    src = a.k + t * a.ldk + static_cast<int64_t>(h - a.q_heads) * a.head_dim;
    dst = a.k_out + t * a.ldko + static_cast<int64_t>(h - a.q_heads) * a.head_dim;
  }
}

// A workgroup takes a token. A unit is 8 pairs of halves (two 16-byte words), 4 pairs of neighbours or 8
// elements behind the rotated ones (one word); with VEC false, for heads that do not start on words, one
// pair or one element (8192 tokens of 24 heads of 128 at an odd address 26 us instead of 17; of 80, 38 of
// them turned, 30, where the bytes take 14). `copy`: the elements behind the rotated ones are
// written too (not where a call rotates in place). A token whose position is outside [0, max_positions) is
// copied bit by bit, or in place left alone.
template <bool INTER, bool VEC>
__global__ void __launch_bounds__(kThreads) rope_angles_kernel(RopeArgs a, int copy) {
  __shared__ float2 angle[kMaxPairs];  // (cos, sin) times the gain
  constexpr int W = VEC ? 8 : 1;       // elements of a word
  const int pairs = a.rotary / 2;
  const int rot_units = VEC ? (INTER ? a.rotary / 8 : pairs / 8) : pairs;
  const int units = rot_units + (copy ? (a.head_dim - a.rotary) / W : 0);  // of a head
  const int64_t t = blockIdx.x;
  const int64_t pos = a.positions[t];
  if (pos < 0 || pos >= a.max_positions) {  // (the whole workgroup's)
    const int words = a.head_dim / W;  // of a head
    for (int u = threadIdx.x; copy && u < a.heads * words; u += kThreads) {
      const int at = (u % words) * W;
      const bf16_t* src;
      bf16_t* dst;
      head_at(a, t, u / words, src, dst);
      if constexpr (VEC) *reinterpret_cast<uint4*>(dst + at) = *reinterpret_cast<const uint4*>(src + at);
      else dst[at] = src[at];
    }
    return;
  }
  for (int i = threadIdx.x; i < pairs; i += kThreads) {
    const float2 sc = sincos_turns(static_cast<uint64_t>(pos) * a.turns[i]);
    angle[i] = make_float2(sc.y * a.gain, sc.x * a.gain);
  }
  __syncthreads();
  const int total = a.heads * units;
  for (int u = threadIdx.x; u < total; u += kThreads) {
    const int head = u / units, i = u % units;
    const bf16_t* src;
    bf16_t* dst;
    head_at(a, t, head, src, dst);
    if (i >= rot_units) {
      const int at = a.rotary + (i - rot_units) * W;
      if constexpr (VEC) *reinterpret_cast<uint4*>(dst + at) = *reinterpret_cast<const uint4*>(src + at);
      else dst[at] = src[at];
    } else if constexpr (!VEC) {
      const int x = INTER ? 2 * i : i, y = INTER ? 2 * i + 1 : pairs + i;
      float o1, o2;
      rope_pair(bf16_to_f32(src[x]), bf16_to_f32(src[y]), angle[i].x, angle[i].y, o1, o2);
      dst[x] = f32_to_bf16(o1);
      dst[y] = f32_to_bf16(o2);
    } else if constexpr (INTER) {
      float x[8], o[8];
      load8(*reinterpret_cast<const uint4*>(src + 8 * i), x);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        rope_pair(x[2 * e], x[2 * e + 1], angle[4 * i + e].x, angle[4 * i + e].y, o[2 * e], o[2 * e + 1]);
      *reinterpret_cast<uint4*>(dst + 8 * i) = store8(o);
    } else {
      float x[8], y[8], o1[8], o2[8];
      load8(*reinterpret_cast<const uint4*>(src + 8 * i), x);
      load8(*reinterpret_cast<const uint4*>(src + pairs + 8 * i), y);
#pragma unroll
      for (int e = 0; e < 8; ++e) rope_pair(x[e], y[e], angle[8 * i + e].x, angle[8 * i + e].y, o1[e], o2[e]);
      *reinterpret_cast<uint4*>(dst + 8 * i) = store8(o1);
      *reinterpret_cast<uint4*>(dst + pairs + 8 * i) = store8(o2);
    }
  }
}

}  // namespace
}  // namespace sid

using namespace sid;

extern "C" int sid_rope_rotate(const void* q, int64_t ldq, const void* k, int64_t ldk,
                               const int64_t* positions, const uint64_t* turns, float gain,
                               int rotary_dim, int interleaved, int64_t num_tokens,
                               int num_q_heads, int num_kv_heads, int head_dim,
                               int64_t max_positions, void* q_out, int64_t ldq_out, void* k_out,
                               int64_t ldk_out, void* stream) {
  const char* name = "rope_rotate";
  SID_REQUIRE(num_tokens >= 0, "%s: negative token count %lld", name, (long long)num_tokens);
  if (num_tokens == 0) return SID_OK;
  SID_REQUIRE(num_q_heads >= 0 && num_kv_heads >= 0 && num_q_heads <= 65536 &&
                  num_kv_heads <= 65536 && num_q_heads + num_kv_heads > 0,
              "%s: bad head counts %d, %d", name, num_q_heads, num_kv_heads);
  SID_REQUIRE(positions && turns && (num_q_heads == 0 || (q && q_out)) &&
                  (num_kv_heads == 0 || (k && k_out)),
              "%s: null pointer", name);
  SID_REQUIRE(head_dim > 0 && head_dim <= 2 * kMaxPairs, "%s: head_dim must be at most %d, got %d",
              name, 2 * kMaxPairs, head_dim);
  SID_REQUIRE(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim,
              "%s: rotary_dim %d must be even and at most head_dim %d", name, rotary_dim, head_dim);
  const int64_t rq = static_cast<int64_t>(num_q_heads) * head_dim;
  const int64_t rk = static_cast<int64_t>(num_kv_heads) * head_dim;
  SID_REQUIRE(ldq >= rq && ldq_out >= rq && ldk >= rk && ldk_out >= rk,
              "%s: a row stride is less than a row", name);
  SID_REQUIRE((q != q_out || ldq == ldq_out) && (k != k_out || ldk == ldk_out),
              "%s: in place, the row strides must be the same", name);
  SID_REQUIRE(num_tokens < (1ll << 24), "%s: too many tokens", name);  // (2^32 threads)
  const bool in_place = (num_q_heads == 0 || q == q_out) && (num_kv_heads == 0 || k == k_out);
  // Words of 16 bytes where every piece of a head starts on one.
  auto word = [](const void* p, int64_t ld, int heads) {
    return heads == 0 || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0);
  };
  const bool vec = head_dim % 8 == 0 && rotary_dim % (interleaved ? 8 : 16) == 0 &&
                   word(q, ldq, num_q_heads) && word(q_out, ldq_out, num_q_heads) &&
                   word(k, ldk, num_kv_heads) && word(k_out, ldk_out, num_kv_heads);
  const RopeArgs a{(const bf16_t*)q, (const bf16_t*)k, (bf16_t*)q_out, (bf16_t*)k_out, ldq, ldk,
                   ldq_out, ldk_out, positions, turns, max_positions, gain, rotary_dim,
                   head_dim, num_q_heads, num_q_heads + num_kv_heads};
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)num_tokens), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), a, in_place ? 0 : 1);
    return check_launch(name);
  };
  if (vec) return interleaved ? go(rope_angles_kernel<true, true>) : go(rope_angles_kernel<false, true>);
  return interleaved ? go(rope_angles_kernel<true, false>) : go(rope_angles_kernel<false, false>);
}
