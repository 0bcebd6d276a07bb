// Rotary positions of the LLM's query and key heads, with the store of k and v
// into the paged caches (include/dllm.h, dllm_rotary).
//
// Each of the rot_dim / 2 pairs (a, b) of a head turns by t = position * w_i:
//   a' = f (a cos t - b sin t),  b' = f (b cos t + a sin t)
// with the pair (d, d + rot_dim / 2) in the half layout and (2d, 2d + 1) in the
// interleaved one; dims past rot_dim are copied.  w_i comes in turns per
// position as a 64-bit binary fraction, so the angle modulo one turn is one
// wrapping 64-bit multiplication, off by at most |position| * 2^-65 turns, of
// which the upper 32 bits are used (another 2^-32): a 32-bit float angle is off by
// 0.06 rad at position 10^6.  What is left of a turn is split into a quarter
// (exact) and an eighth-turn remainder for sincospif.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace dfm {

constexpr int RO_THREADS = 256;

struct RotaryParams {
  const unsigned long long* turns;   // [rot / 2]
  const int* positions;              // [tokens]
  const void* q;
  void* q_out;
  const void* k;
  const void* v;
  void* k_cache;
  void* v_cache;
  const int* slots;                  // [tokens], null without the store
  uint32_t* err;
  long long q_ts, q_hs, o_ts, o_hs, k_ts, k_hs, v_ts, v_hs;   // element strides
  long long num_slots;
  int tokens, heads, kv_heads, D, rot;
  float factor;
  bool copy_tail;                    // q_out is not q: its unrotated dims are written too
  FastDiv by_token, by_lanes, by_pairs;   // items of a token, lanes of a head, pairs of a head
};

DFM_DEV void rotary_sincos(unsigned long long w, int pos, float f, float& c, float& s) {
  const uint32_t t = static_cast<uint32_t>((static_cast<unsigned long long>(static_cast<long long>(pos)) * w) >> 32);
  const uint32_t quarter = (t + 0x20000000u) >> 30;
  const int rest = static_cast<int>(t - (quarter << 30));
  float s0, c0;
  sincospif(static_cast<float>(rest) * 4.656612873077393e-10f, &s0, &c0);   // 2^-31: half turns
  const float a = (quarter & 1) ? -s0 : c0, b = (quarter & 1) ? c0 : s0;
  c = ((quarter & 2) ? -a : a) * f;
  s = ((quarter & 2) ? -b : b) * f;
}

template <typename T>
DFM_DEV float ro_load(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}
template <typename T>
DFM_DEV T ro_store(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else return __float2bfloat16(x);
}

// Where head h of token t is read and written: q heads, then k, then v.
template <typename T>
struct RotaryHead {
  const T* src;
  T* dst;
  bool turn;     // rotated (q, k) or copied (v)
  bool tail;     // its unrotated dims are written
};

template <typename T>
DFM_DEV RotaryHead<T> rotary_head(const RotaryParams& p, int t, int h, int slot) {
  RotaryHead<T> r;
  if (h < p.heads) {
    r.src = static_cast<const T*>(p.q) + t * p.q_ts + h * p.q_hs;
    r.dst = static_cast<T*>(p.q_out) + t * p.o_ts + h * p.o_hs;
    r.turn = true;
    r.tail = p.copy_tail;
    return r;
  }
  h -= p.heads;
  r.turn = h < p.kv_heads;
  if (!r.turn) h -= p.kv_heads;
  const void* base = r.turn ? p.k : p.v;
  void* cache = r.turn ? p.k_cache : p.v_cache;
  r.src = static_cast<const T*>(base) + t * (r.turn ? p.k_ts : p.v_ts) + h * (r.turn ? p.k_hs : p.v_hs);
  r.dst = slot < 0 ? nullptr
                   : static_cast<T*>(cache) + (static_cast<long long>(slot) * p.kv_heads + h) * p.D;
  r.tail = true;
  return r;
}

// The token's cache slot, or -1 for none; one past the cache is reported.
DFM_DEV int rotary_slot(const RotaryParams& p, int t, bool report) {
  if (!p.slots) return -1;
  const int slot = p.slots[t];
  if (slot < p.num_slots) return slot < 0 ? -1 : slot;
  if (report) atomicOr(p.err, DFM_DEV_ERR_PAGE);
  return -1;
}

// Any layout: one thread per (token, head, pair of elements).
template <typename T, bool INTER>
__global__ void __launch_bounds__(RO_THREADS) llm_rotary_scalar_kernel(RotaryParams p) {
  pdl_trigger();
  pdl_wait();
  const int per_head = (p.D + 1) / 2, heads = p.heads + (p.slots ? 2 * p.kv_heads : 0);
  const long long idx = static_cast<long long>(blockIdx.x) * RO_THREADS + threadIdx.x;
  if (idx >= static_cast<long long>(p.tokens) * heads * per_head) return;
  const int e = static_cast<int>(idx % per_head);
  const long long th = idx / per_head;
  const int h = static_cast<int>(th % heads), t = static_cast<int>(th / heads);
  const int slot = h >= p.heads ? rotary_slot(p, t, e == 0) : 0;
  const RotaryHead<T> r = rotary_head<T>(p, t, h, slot);
  if (!r.dst) return;
  const int half = p.rot / 2;
  if (r.turn && e < half) {
    const int a = INTER ? 2 * e : e, b = INTER ? 2 * e + 1 : e + half;
    float c, s;
    rotary_sincos(p.turns[e], p.positions[t], p.factor, c, s);
    const float x = ro_load(r.src[a]), y = ro_load(r.src[b]);
    r.dst[a] = ro_store<T>(x * c - y * s);
    r.dst[b] = ro_store<T>(y * c + x * s);
    return;
  }
  if (!r.tail) return;
  // pair e holds elements 2e and 2e + 1; past the rotated dims these are copied
  for (int d = 2 * e; d < 2 * e + 2 && d < p.D; ++d) r.dst[d] = r.src[d];
}

// Whole 16-byte vectors.  A block takes TB tokens: its threads first compute the
// tokens' cosines and sines, one pair each, into shared memory (threads that
// compute those of their own vectors: 33 us instead of 27 at the size below), then
// turn items of VP pairs of a head: lane l of D / (2 VP) has pairs [l VP, (l + 1) VP)
// or, past the rotated dims, copies two vectors.  A thread's first item is loaded
// before the angles are computed.  Bound by HBM and the latency of a block's
// three dependent loads: 16384 tokens of 12 + 2 + 2 heads of 128 (134 MB) in 27.2 us,
// 4.9 TB/s.  Two items a thread need 64 registers instead of 40: 30.4 us.
constexpr int RO_MAX_PAIRS = 256;    // of a head in the table

template <typename T, bool INTER, int TB>
__global__ void __launch_bounds__(RO_THREADS, 6) llm_rotary_kernel(RotaryParams p) {
  constexpr int VP = 16 / sizeof(T);
  __shared__ float4 table[TB][RO_MAX_PAIRS / 2];   // cosine and sine of two pairs: read 16 bytes at a time
  pdl_trigger();
  pdl_wait();
  const int half = p.rot / 2, heads = p.heads + (p.slots ? 2 * p.kv_heads : 0);
  const int lanes = p.D / (2 * VP), per_token = heads * lanes;
  const int t0 = blockIdx.x * TB, tokens = min(TB, p.tokens - t0), items = tokens * per_token;
  RotaryHead<T> r;
  int t, a, b, l;        // token of the block, the two vectors' elements, the lane
  bool on, turn;
  uint4 va, vb;
  auto load = [&](int item) {
    on = item < items;
    if (!on) return;
    t = TB > 1 ? p.by_token(item) : 0;
    const int rest = item - t * per_token, h = p.by_lanes(rest);
    l = rest - h * lanes;
    r = rotary_head<T>(p, t0 + t, h, h >= p.heads ? rotary_slot(p, t0 + t, l == 0) : 0);
    turn = r.turn && l * VP < half;
    on = r.dst && (turn || r.tail);
    if (!on) return;
    a = turn && !INTER ? l * VP : 2 * l * VP;
    b = turn && !INTER ? a + half : a + VP;
    va = *reinterpret_cast<const uint4*>(r.src + a);
    vb = *reinterpret_cast<const uint4*>(r.src + b);
  };
  load(threadIdx.x);
  for (int i = threadIdx.x; i < tokens * half; i += RO_THREADS) {
    const int tok = TB > 1 ? p.by_pairs(i) : 0, e = i - tok * half;
    float c, s;
    rotary_sincos(p.turns[e], p.positions[t0 + tok], p.factor, c, s);
    reinterpret_cast<float2*>(table[tok])[e] = make_float2(c, s);
  }
  __syncthreads();
  for (int item = threadIdx.x; item < items; item += RO_THREADS) {
    if (item >= RO_THREADS) load(item);
    if (!on) continue;
    if (turn) {
      T* x = reinterpret_cast<T*>(&va);
      T* y = reinterpret_cast<T*>(&vb);
      const float4* cs = &table[t][l * VP / 2];
#pragma unroll
      for (int i = 0; i < VP; i += 2) {
        const float4 c = cs[i / 2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          // half layout: pair n is (x[n], y[n]); interleaved: elements 2n and 2n + 1 of x|y
          const int n = i + k;
          T* xp = INTER ? (2 * n < VP ? x + 2 * n : y + 2 * n - VP) : x + n;
          T* yp = INTER ? xp + 1 : y + n;
          const float u = ro_load(*xp), w = ro_load(*yp), co = k ? c.z : c.x, si = k ? c.w : c.y;
          *xp = ro_store<T>(u * co - w * si);
          *yp = ro_store<T>(w * co + u * si);
        }
      }
    }
    *reinterpret_cast<uint4*>(r.dst + a) = va;
    *reinterpret_cast<uint4*>(r.dst + b) = vb;
  }
}

}  // namespace dfm
