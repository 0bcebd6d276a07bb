// Rotary positions of the LLM's query and key heads, with the store of k and v
// into the paged caches (include/dllm.h, dllm_rotary).
//
// Each of the rot_dim / 2 pairs (a, b) of a head turns by t = position * w_i:
//   a' = f (a cos t - b sin t),  b' = f (b cos t + a sin t)
// with the pair (d, d + rot_dim / 2) in the half layout and (2d, 2d + 1) in the
// interleaved one; dims past rot_dim are copied.  w_i comes in turns per
// position as a 64-bit binary fraction, so the angle modulo one turn is one
// wrapping 64-bit multiplication, off by at most |position| * 2^-65 turns: a
// 32-bit float angle is off by 0.06 rad at position 10^6.  What is left of a
// turn is split into a quarter (exact) and an eighth-turn remainder for
// sincospif.
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

// Whole 16-byte vectors: VP pairs a thread, over HG heads of one token.  A
// token takes D / (2 VP) lanes; lane l turns pairs [l VP, (l + 1) VP) or, past
// the rotated dims, copies two vectors.  All HG heads' loads are issued before
// the first result is written.
template <typename T, bool INTER, int HG>
__global__ void __launch_bounds__(RO_THREADS) llm_rotary_kernel(RotaryParams p) {
  constexpr int VP = 16 / sizeof(T);
  pdl_trigger();
  pdl_wait();
  const int lanes = p.D / (2 * VP), heads = p.heads + (p.slots ? 2 * p.kv_heads : 0);
  const int groups = (heads + HG - 1) / HG;
  const long long idx = static_cast<long long>(blockIdx.x) * RO_THREADS + threadIdx.x;
  if (idx >= static_cast<long long>(p.tokens) * groups * lanes) return;
  const int l = static_cast<int>(idx % lanes);
  const long long tg = idx / lanes;
  const int h0 = static_cast<int>(tg % groups) * HG, t = static_cast<int>(tg / groups);
  const int half = p.rot / 2;
  const bool turning = l * VP < half;
  // the two vectors of this lane, in elements of the head: rotated pairs, and
  // the copy of a head that is not rotated (or of dims past rot_dim)
  const int ta = INTER ? 2 * l * VP : l * VP, tb = INTER ? ta + VP : ta + half;
  const int ca = 2 * l * VP, cb = ca + VP;
  const int slot = h0 + HG > p.heads ? rotary_slot(p, t, l == 0) : 0;
  uint4 va[HG], vb[HG];
#pragma unroll
  for (int j = 0; j < HG; ++j) {
    if (h0 + j >= heads) continue;
    const RotaryHead<T> r = rotary_head<T>(p, t, h0 + j, slot);
    const bool turn = r.turn && turning;
    if (!r.dst || !(turn || r.tail)) continue;
    va[j] = *reinterpret_cast<const uint4*>(r.src + (turn ? ta : ca));
    vb[j] = *reinterpret_cast<const uint4*>(r.src + (turn ? tb : cb));
  }
  float c[VP], s[VP];
  if (turning && h0 < p.heads + p.kv_heads) {
    const int pos = p.positions[t];
#pragma unroll
    for (int i = 0; i < VP; ++i) rotary_sincos(p.turns[l * VP + i], pos, p.factor, c[i], s[i]);
  }
#pragma unroll
  for (int j = 0; j < HG; ++j) {
    if (h0 + j >= heads) continue;
    const RotaryHead<T> r = rotary_head<T>(p, t, h0 + j, slot);
    const bool turn = r.turn && turning;
    if (!r.dst || !(turn || r.tail)) continue;
    if (turn) {
      T* a = reinterpret_cast<T*>(&va[j]);
      T* b = reinterpret_cast<T*>(&vb[j]);
#pragma unroll
      for (int i = 0; i < VP; ++i) {
        // half layout: pair i is (a[i], b[i]); interleaved: elements 2i and 2i + 1 of a|b
        T* xp = INTER ? (2 * i < VP ? a + 2 * i : b + 2 * i - VP) : a + i;
        T* yp = INTER ? xp + 1 : b + i;
        const float x = ro_load(*xp), y = ro_load(*yp);
        *xp = ro_store<T>(x * c[i] - y * s[i]);
        *yp = ro_store<T>(y * c[i] + x * s[i]);
      }
    }
    *reinterpret_cast<uint4*>(r.dst + (turn ? ta : ca)) = va[j];
    *reinterpret_cast<uint4*>(r.dst + (turn ? tb : cb)) = vb[j];
  }
}

}  // namespace dfm
