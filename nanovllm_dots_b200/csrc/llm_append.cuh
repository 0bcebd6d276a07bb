// Append attention of the LLM backbone: new tokens of many sequences over the
// paged K/V cache that already holds them (include/dllm.h,
// dllm_append_attention).
//
// Row (token j of sequence i, query head h) sees the keys of one interval
// [lo, hi) (causal, sliding window, bidirectional prefix and document masks all
// are one) or, when a tree of drafted tokens is verified, the history [0, base)
// and the drafted keys in the token's 64-bit mask:
//   s_k = cap tanh(scale q.k / cap) - slope_h |p - k|     (cap and slope optional)
//   o = sum_k exp(s_k - m) v_k / sum_k exp(s_k - m),  zeros if the row sees no key.
//
// Work.  The G query heads of a kv head are packed with the tokens into rows,
// row = token * G + head, RT = 128 / G tokens to a 128-row tile, so K and V are
// read once for all of them and single tokens, trees and prompts take the same
// path.  A unit is up to two row tiles of a sequence; its keys are taken in
// tiles of 128, newest first (the tiles with masks first, and with a distance
// bias the largest scores first).  The units of every kv head, each a fixed cost
// and its key tiles, form one line that is cut into equal shares for the
// persistent CTAs: a unit whose keys fall into several shares leaves unnormalised
// partials that llm_append_combine_kernel adds up in the order of the shares.
//
// One CTA per SM, 12 warps: two softmax warpgroups (a thread is a row), a TMA
// warp, an MMA warp and two warps that look after V.  Each softmax warpgroup
// works on a stream of its own (score tile S in TMEM, overwritten by the
// probabilities P, and the accumulator O): the two row tiles of a wide unit
// over every key tile, or the one row tile of a narrow unit over the even and
// the odd key tiles, merged at the end.  One stream's softmax runs under the
// other's products:
//   S[128 x 128] = Q K^T      (Q and K from shared memory)
//   O[128 x D]  += P V        (P from TMEM, V from shared memory)
//
// What bounds it.  Single tokens and small trees: HBM, at its rate while the tiles
// stream (64 single tokens over 4000 positions of 4 x 128 dims: 99 us, 5.5 TB/s), plus
// the fixed way in (3.5 us from the start to the first scores) and out (join 4.5 us).
// Two full row tiles: a stream's chain of maximum (750 clocks), probabilities (1500)
// and the products of P and of the next scores (1250 of latency and of the other
// stream's): 3500 clocks a key tile, of which the tensor cores are busy 2048 with
// D = 128.  8192 tokens behind 8192: 526 us, 1.17 PFLOP/s (605 us and 1.02 under the
// power cap; the same loads and products without a softmax 440).  With D = 128 all 512
// TMEM columns are taken (S, S, O, O), so scores cannot be computed ahead of P, which
// the 128 columns left with D = 64 would allow; key tiles of 64 in two buffers, which
// could, take the tensor cores twice as long a score (676 us); two threads a row
// instead of one: 568.
//
// P is rounded to the type of V, which the product asks of both (half a step, relative
// to each probability); scores, maxima, sums and O are fp32, and the sum takes P
// before its rounding.  For given lengths a row's result depends on its own query and
// the keys that it sees, bit for bit: what a warp decides together only chooses the
// way there.
//
// Keys nobody in the unit may see are not loaded (their pages may be gone) and
// their rows of V are set to zero.  In a tile with masks, an infinity or a NaN in a
// visible row of V is set to zero as well (0 * inf in the product would reach
// every row) and the key noted: the rows that see it add it to their output at
// the end, at its own dim.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace dfm {

constexpr int AP_KT = 128;          // keys per tile
constexpr int AP_ROWS = 128;        // rows per tile (TMEM lanes)
constexpr int AP_SOFT_WARPS = 8;
constexpr int AP_THREADS = 32 * (AP_SOFT_WARPS + 4);
constexpr int AP_PLAN_THREADS = 1024;
constexpr int AP_COMBINE_THREADS = 256, AP_COMBINE_BLOCKS = 3;   // blocks to an SM
constexpr int AP_MAX_CTAS = 256;    // most SMs the shares go to
constexpr int AP_NEAR_SEQS = 256, AP_NEAR_UNITS = 512;   // what a CTA plans by itself
constexpr int AP_NEAR_FIRST = 64;   // units, where every token has bounds of its own (6000 packed
                                    // tokens: 72 us instead of 75 with a kernel of its own)
// What a unit costs besides its tiles (its first loads, the masked tiles, its rows'
// way out: 4000 to 8000 clocks), in half tiles of a wide unit (1800 clocks).  With
// shares of equal tiles alone, CTAs with many short units ended last: a chunked
// prefill of 24 sequences took 62.0 us instead of 49.2, 64 single tokens 30.4 instead
// of 28.7, 64 small trees 30.1 instead of 28.3; 2 / 4 and 3 / 4 are equal, 1 / 3 and
// 3 / 6 slower.
constexpr int AP_NARROW_COST = 3, AP_WIDE_COST = 4;
constexpr int AP_MIN_SHARE = 2;     // smallest share of the line (a wide unit's key tile counts 2)
// The running maximum of a row is raised only when a score passes it by this
// much (log2 units): probabilities then reach 2^8, exact in fp32 and within
// fp16's range, and O is seldom rescaled.
constexpr float AP_TAU = 8.0f;
// Of AP_EXP_OF pairs of exponentials, AP_EXP_POLY go to the fp32 pipe: the special
// function unit takes 8 clocks a warp's exponential.  A quarter is the fastest of
// none, a quarter, a third and a half.
constexpr int AP_EXP_POLY = 1, AP_EXP_OF = 4;

struct __align__(16) ApUnit {
  int seq, t0, ntok, row0;          // tokens [t0, t0 + ntok) of the sequence; row0: its first in q
  int lo, hi, fmin, fmax;           // union of the rows' keys; tiles inside [fmin, fmax) have no mask
  int base, m, pre, at;             // position of token 0; the sequence's tokens and prefix; place in the line
  DFM_DEV void keys(const ApUnit& o) { lo = o.lo, hi = o.hi, fmin = o.fmin, fmax = o.fmax; }
  DFM_DEV int tiles() const { return hi > lo ? (hi + AP_KT - 1) / AP_KT - lo / AP_KT : 0; }
  DFM_DEV int lead(int rt) const { return ntok > rt ? AP_WIDE_COST : AP_NARROW_COST; }
  DFM_DEV int cost(int rt) const { return lead(rt) + (tiles() << (ntok > rt)); }   // a wide unit's tile counts 2
};
static_assert(sizeof(ApUnit) == 48, "unit record");

struct ApHead {                     // the plan's header
  int line, share, units, pad;      // length of one kv head's line, of one CTA's share
};

struct ApCut {                      // the unit that the end of a share cuts
  int row, ntok, kv;                // its first token's row in q
  int last;                         // last share it reaches into; -1: no unit of this share is cut
};

struct ApParams {
  const int* cu;                    // [n + 1]
  const int* ctx;                   // [n]
  const int* bt;                    // [n][max_blocks]
  const int* prefix;                // [n] or null
  const int* first;                 // [tokens] or null
  const unsigned long long* tree;   // [tokens] or null
  const float* slopes;              // [H] or null
  const void* v;                    // the V cache, for its special values
  void* out;                        // [tokens][H][D]
  uint32_t* err;
  ApHead* head;                     // head .. start: of the plan kernel, unused with near_plan
  ApUnit* units;
  int* ubase;                       // [n]
  int* start;                       // [ctas + 1] unit at the start of each share
  ApCut* cuts;                      // [ctas]
  float* part_o;                    // [ctas][2][2][D / 8][128][8]
  float2* part_ml;                  // [ctas][2][2][128]
  void* special;                    // ApSpecial<D> [ctas][2 streams][128]
  int tokens, n, H, KVH, G, RT, max_units, ctas, near_plan;
  int num_blocks, block_size, max_blocks, box_rows;
  int causal, window;
  FastDiv by_g, by_unit, by_ctas, by_block;   // G, 2 RT, ctas, block_size
  float scale_log2;                 // scale * log2(e)
  // With a cap (cap_a 0: none): cap_a = scale / cap, cap_b its inverse, cap_in =
  // 2 log2(e) cap_a and tanh's polynomial in powers of cap_a, taken up to |q.k| = cap_hot.
  float cap_a, cap_b, cap_in, cap_hot, cap_q[3];
  float cap_y[4];                   // the polynomial times scale_log2
};

// ---------------------------------------------------------------- plan
// Sums of two values over the threads before this one and over all of the
// block's kWarps warps.
template <int kWarps>
DFM_DEV int2 block_scan(int2 v, int2* warp_sums, int2& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, x.x, o), b = __shfl_up_sync(0xffffffffu, x.y, o);
    if (lane >= o) {
      x.x += a;
      x.y += b;
    }
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int2 w = lane < kWarps ? warp_sums[lane] : make_int2(0, 0);
  const bool mine = lane < warp;
  const int2 before = make_int2(__reduce_add_sync(0xffffffffu, mine ? w.x : 0),
                                __reduce_add_sync(0xffffffffu, mine ? w.y : 0));
  total = make_int2(__reduce_add_sync(0xffffffffu, w.x), __reduce_add_sync(0xffffffffu, w.y));
  __syncthreads();
  return make_int2(before.x + x.x - v.x, before.y + x.y - v.y);
}

// Rows [s0, s0 + m) of sequence i; whether they make sense.
DFM_DEV bool ap_rows(const ApParams& p, int i, int& s0, int& m) {
  s0 = p.cu[i];
  const int s1 = p.cu[i + 1];
  m = s1 - s0;
  return s0 >= 0 && s1 >= s0 && s1 <= p.tokens;
}

// Whether ctx cached positions with m new tokens make sense.
DFM_DEV bool ap_length(const ApParams& p, int m, int ctx) {
  return ctx >= m && ctx <= static_cast<long long>(p.max_blocks) * p.block_size && !(p.tree && m > 64);
}

// [lo, hi) of new token j (row s0 + j of q) without a tree; pre: the sequence's prefix.
DFM_DEV void ap_keys(const ApParams& p, int s0, int j, int base, int ctx, int pre, int& lo, int& hi) {
  const int pos = base + j;
  hi = p.causal ? max(pos + 1, min(pre, ctx)) : ctx;
  lo = p.window ? max(0, pos + 1 - p.window) : 0;
  if (p.first) lo = max(lo, p.first[s0 + j]);
}

// The unit at token t0 of a sequence; with per-token bounds (p.first) lo .. fmax
// are the caller's.
DFM_DEV ApUnit ap_unit(const ApParams& p, int seq, int s0, int m, int ctx, int pre, int t0) {
  ApUnit f;
  f.seq = seq;
  f.t0 = t0;
  f.ntok = min(2 * p.RT, m - t0);
  f.row0 = s0;
  f.base = ctx - m;
  f.m = m;
  f.pre = pre;
  f.lo = f.hi = f.fmax = 0;
  f.fmin = 0x7fffffff;
  f.at = 0;
  if (ap_length(p, m, ctx)) {
    if (p.tree) {
      f.hi = ctx;
      f.fmin = 0;
      f.fmax = f.base;
    } else if (!p.first) {   // the ends of the interval rise with the token
      ap_keys(p, s0, t0, f.base, ctx, pre, f.lo, f.fmax);
      ap_keys(p, s0, t0 + f.ntok - 1, f.base, ctx, pre, f.fmin, f.hi);
    }
  }
  return f;
}

// With bounds of every token's own: lo .. fmax of the unit at token t0, by a warp.
DFM_DEV int4 ap_bounds(const ApParams& p, int s0, int m, int ctx, int pre, int t0) {
  const int last = min(m, t0 + 2 * p.RT) - 1;
  int lo = 0x7fffffff, hi = 0, fmin = 0, fmax = 0x7fffffff;
  for (int j0 = t0 + (threadIdx.x & 31); j0 - 31 <= last; j0 += 32 * 4) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {   // past the end, the last token again
      int l, h;
      ap_keys(p, s0, min(j0 + 32 * x, last), ctx - m, ctx, pre, l, h);
      if (l < h) {
        lo = min(lo, l);
        hi = max(hi, h);
      }
      fmin = max(fmin, l);
      fmax = min(fmax, h);
    }
  }
  return make_int4(__reduce_min_sync(0xffffffffu, lo), __reduce_max_sync(0xffffffffu, hi),
                   __reduce_max_sync(0xffffffffu, fmin), __reduce_min_sync(0xffffffffu, fmax));
}

DFM_DEV int ap_share(const ApParams& p, int line) {
  return max(AP_MIN_SHARE, p.by_ctas(line * p.KVH + p.ctas - 1));
}

// The plan of a batch small enough for every CTA to make it in its own shared
// memory: that takes about a microsecond, a kernel of its own three.
struct ApNear {
  ApUnit units[AP_NEAR_UNITS];
  int2 sums[AP_THREADS / 32];
  int line, count, share;
  int first, kv, off;   // where this CTA's share starts: unit, kv head, place in the unit

  // Scratch of make(), which is over before the memory is used for anything else.
  struct Seqs {
    int s0[AP_NEAR_SEQS], m[AP_NEAR_SEQS], ctx[AP_NEAR_SEQS], pre[AP_NEAR_SEQS], ubase[AP_NEAR_SEQS];
  };

  // All AP_THREADS threads.
  DFM_DEV void make(const ApParams& p, Seqs& q) {
    const int t = threadIdx.x;
    int c = 0, cost = 0;
    ApUnit f;
    if (t < p.n) {
      int s, k;
      const bool rows = ap_rows(p, t, s, k);
      const int x = p.ctx[t], pr = p.prefix ? p.prefix[t] : 0;
      if (rows) c = min(p.by_unit(k + 2 * p.RT - 1), AP_NEAR_UNITS);
      if (blockIdx.x == 0 && !(rows && ap_length(p, k, x))) atomicOr(p.err, DFM_DEV_ERR_LEN);
      if (c > 0) {
        f = ap_unit(p, t, s, k, x, pr, 0);
        cost = f.cost(p.RT);
      }
      q.s0[t] = s;
      q.m[t] = k;
      q.ctx[t] = x;
      q.pre[t] = pr;
    }
    // units, and above bit 20 the sequences that have some; places if each has one
    int2 all;
    const int2 before = block_scan<AP_THREADS / 32>(make_int2(c | (c > 0) << 20, cost), sums, all);
    int u = before.x & 0xfffff, place = before.y, total = all.x & 0xfffff;
    const bool several = p.first || total != all.x >> 20;
    if (t < p.n) q.ubase[t] = u;
    if (total > p.max_units) {   // rows of overlapping sequences
      if (blockIdx.x == 0 && t == 0) atomicOr(p.err, DFM_DEV_ERR_LEN);
      total = p.max_units;
    }
    auto start = [&](bool mine) {   // the share starts in this thread's unit u
      const int sh = ap_share(p, all.y), g = blockIdx.x * sh;
      if (t == 0) {
        line = all.y;
        count = total;
        share = sh;
      }
      if (!mine || g >= all.y * p.KVH) return;
      const int h = g / all.y, o = g - h * all.y - place;
      if (o < 0 || o >= cost) return;
      first = u;
      kv = h;
      off = o;
    };
    if (!several) {              // a unit to a sequence
      const bool mine = c > 0 && u < total;
      if (mine) {
        f.at = place;
        units[u] = f;
      }
      start(mine);
    } else {
      __syncthreads();
      auto seq_of = [&](int v) {   // the last sequence with ubase <= v (one without units shares the next one's)
        int a = 0, b = p.n - 1;
        while (a < b) {
          const int mid = (a + b + 1) >> 1;
          if (q.ubase[mid] <= v) a = mid; else b = mid - 1;
        }
        return a;
      };
      if (p.first) {
        for (u = t >> 5; u < total; u += AP_THREADS / 32) {
          const int a = seq_of(u);
          if (!ap_length(p, q.m[a], q.ctx[a])) continue;
          const int4 k = ap_bounds(p, q.s0[a], q.m[a], q.ctx[a], q.pre[a], (u - q.ubase[a]) * 2 * p.RT);
          if ((t & 31) == 0) *reinterpret_cast<int4*>(&units[u].lo) = k;
        }
        __syncthreads();
      }
      all.y = 0;
#pragma unroll 1
      for (int u0 = 0; u0 < total; u0 += AP_THREADS) {
        u = u0 + t;
        cost = 0;
        if (u < total) {
          const int a = seq_of(u);
          f = ap_unit(p, a, q.s0[a], q.m[a], q.ctx[a], q.pre[a], (u - q.ubase[a]) * 2 * p.RT);
          if (p.first && ap_length(p, f.m, q.ctx[a])) f.keys(units[u]);
          cost = f.cost(p.RT);
        }
        int2 sum;
        place = all.y + block_scan<AP_THREADS / 32>(make_int2(cost, 0), sums, sum).x;
        if (u < total) {
          f.at = place;
          units[u] = f;
        }
        all.y += sum.x;
      }
      __syncthreads();
      for (u = t; u < total; u += AP_THREADS) {
        place = units[u].at;
        cost = units[u].cost(p.RT);
        start(true);
      }
      start(false);
    }
    fence_proxy_async_smem();   // the scratch lies where copies will land
    __syncthreads();
  }
};
static_assert(AP_NEAR_SEQS <= AP_THREADS, "a thread to a sequence");

// The plan of larger batches: units, their keys and
// their places in the line, from the device's lengths.  A sequence whose lengths
// make no sense is reported: its rows are written as zeros, or not at all when
// not even they are known.
__global__ void __launch_bounds__(AP_PLAN_THREADS) llm_append_plan_kernel(ApParams p) {
  __shared__ int2 sums[32];
  __shared__ int near[AP_PLAN_THREADS];   // ubase of the first sequences
  constexpr int W = AP_PLAN_THREADS / 32;
  pdl_trigger();
  pdl_wait();
  const int t = threadIdx.x;
  int carry = 0;
  for (int i0 = 0; i0 < p.n; i0 += AP_PLAN_THREADS) {
    const int i = i0 + t;
    int c = 0;
    if (i < p.n) {
      int s0, m;
      const bool rows = ap_rows(p, i, s0, m);
      if (rows) c = p.by_unit(m + 2 * p.RT - 1);
      if (!(rows && ap_length(p, m, p.ctx[i]))) atomicOr(p.err, DFM_DEV_ERR_LEN);
    }
    int2 total;
    const int at = block_scan<W>(make_int2(c, 0), sums, total).x;
    if (i < AP_PLAN_THREADS) near[i] = carry + at;
    else if (i < p.n) p.ubase[i] = carry + at;
    carry += total.x;
  }
  int units = carry;
  if (units > p.max_units) {   // rows of overlapping sequences
    if (t == 0) atomicOr(p.err, DFM_DEV_ERR_LEN);
    units = p.max_units;
  }
  __syncthreads();   // near and ubase, written by this block, are read below
  auto ubase = [&](int i) { return i < AP_PLAN_THREADS ? near[i] : p.ubase[i]; };
  auto seq_of = [&](int u) {   // the last sequence with ubase <= u (one without units shares the next one's)
    int a = 0, b = p.n - 1;
    while (a < b) {
      const int mid = (a + b + 1) >> 1;
      if (ubase(mid) <= u) a = mid; else b = mid - 1;
    }
    return a;
  };
  if (p.first) {   // every token has bounds of its own: a warp to a unit
    for (int u = t >> 5; u < units; u += W) {
      const int a = seq_of(u);
      int s0, m;
      ap_rows(p, a, s0, m);
      const int ctx = p.ctx[a], pre = p.prefix ? p.prefix[a] : 0;
      if (!ap_length(p, m, ctx)) continue;
      const int4 k = ap_bounds(p, s0, m, ctx, pre, (u - ubase(a)) * 2 * p.RT);
      if ((t & 31) == 0) *reinterpret_cast<int4*>(&p.units[u].lo) = k;
    }
    __syncthreads();
  }
  int line = 0;
  for (int u0 = 0; u0 < units; u0 += AP_PLAN_THREADS) {
    const int u = u0 + t;
    ApUnit f;
    int cost = 0;
    if (u < units) {
      const int a = seq_of(u);
      int s0, m;
      ap_rows(p, a, s0, m);
      const int ctx = p.ctx[a];
      f = ap_unit(p, a, s0, m, ctx, p.prefix ? p.prefix[a] : 0, (u - ubase(a)) * 2 * p.RT);
      if (p.first && ap_length(p, m, ctx)) f.keys(p.units[u]);
      cost = f.cost(p.RT);
    }
    int2 total;
    const int at = line + block_scan<W>(make_int2(cost, 0), sums, total).x;
    if (u < units) {
      f.at = at;
      p.units[u] = f;
    }
    line += total.x;
  }
  const int share = ap_share(p, line);
  if (t == 0) {
    p.head->line = line;
    p.head->share = share;
    p.head->units = units;
  }
  // the unit at the start of each share
  for (int u = t; u < units; u += AP_PLAN_THREADS) {
    const ApUnit f = p.units[u];
    for (int kv = 0; kv < p.KVH; ++kv) {
      const int a = kv * line + f.at, b = a + f.cost(p.RT);
      for (int c = (a + share - 1) / share; c * share < b; ++c) p.start[c] = u;
    }
  }
}

// ---------------------------------------------------------------- a CTA's segments
// A segment: key tiles [i0, i1) of a unit (0 is the newest) for one kv head.
struct ApSegment {
  ApUnit f;
  int kv, i0, i1, tiles, top;       // tiles of the whole unit; key tile of i = top - i
  bool narrow;                      // one row tile only
  DFM_DEV bool whole() const { return i0 == 0 && i1 == tiles; }
};

struct ApWalk {
  const ApNear& near;
  int left, line, share, off;       // off: into the unit
  int u, kv, units;

  DFM_DEV ApWalk(const ApParams& p, const ApNear& nr) : near(nr) {
    if (p.near_plan) {
      line = near.line;
      units = near.count;
      share = near.share;
    } else {
      line = p.head->line;
      units = p.head->units;
      share = p.head->share;
    }
    const int all = line * p.KVH, g = blockIdx.x * share;
    left = max(0, min(share, all - g));
    if (left == 0) return;
    if (p.near_plan) {
      u = near.first;
      kv = near.kv;
      off = near.off;
    } else {
      kv = g / line;
      u = p.start[blockIdx.x];
      off = g - kv * line - p.units[u].at;
    }
  }
  // The next segment with work; false at the end of the share.
  DFM_DEV bool next(const ApParams& p, ApSegment& s) {
    while (left > 0) {
      s.f = p.near_plan ? near.units[u] : p.units[u];
      s.kv = kv;
      s.narrow = s.f.ntok <= p.RT;
      const int wide = !s.narrow, lead = s.f.lead(p.RT), cost = s.f.cost(p.RT);
      s.tiles = s.f.tiles();
      s.top = (s.f.hi + AP_KT - 1) / AP_KT - 1;
      const int end = min(off + left, cost);
      s.i0 = (max(0, off - lead) + wide) >> wide;
      s.i1 = min(s.tiles, (max(0, end - lead) + wide) >> wide);
      const bool zero = s.tiles == 0 && off == 0;
      left -= end - off;
      off = end;
      if (end == cost) {
        off = 0;
        if (++u == units) {
          u = 0;
          ++kv;
        }
      }
      if (zero) s.i0 = s.i1 = 0;
      if (zero || s.i1 > s.i0) return true;
    }
    return false;
  }
};

// ---------------------------------------------------------------- shared memory
template <int D>
struct ApSmem {
  static constexpr int BOXES = D / 64;
  // K tiles and V tiles: as many as there is room for (64 single tokens with heads of
  // 64 over 6000 positions: 112 us with 2, 87 with 4).
  static constexpr int RING = D == 64 ? 4 : 2;
  static constexpr int TILE = AP_KT * D * 2;              // one K, V or Q tile
  static constexpr int HALF = AP_KT * 128;                // its 64-dim boxes
  static constexpr int OFF_Q = 0;                         // [2]
  static constexpr int OFF_K = OFF_Q + 2 * TILE;          // [RING]
  static constexpr int OFF_V = OFF_K + RING * TILE;    // [RING]
  static constexpr int OFF_ML = OFF_V + RING * TILE;   // float2 [2 streams][128]
  static constexpr int OFF_NEAR = OFF_ML + 2 * AP_ROWS * 8;
  static constexpr int OFF_BAR = OFF_NEAR + (static_cast<int>(sizeof(ApNear)) + 15) / 16 * 16;
  static constexpr int BYTES = OFF_BAR + 512 + 1024;
};
static_assert(ApSmem<128>::BYTES <= 232448, "one CTA per SM");
static_assert(sizeof(ApNear::Seqs) <= ApSmem<64>::TILE, "the plan's scratch lies on a query tile");

DFM_DEV bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// D(tmem) (+)= A(tmem) * B(smem, MN-major), 16-bit inputs, fp32 accumulate.
DFM_DEV void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                         uint32_t accumulate) {
  const uint32_t z = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}\n" ::"r"(
          d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(z), "r"(z), "r"(z), "r"(z)
      : "memory");
}

// Bounded waits on the SM's clock, which is read in a few cycles (globaltimer is
// not): about a second at the highest clock.
constexpr long long AP_WAIT_CLOCKS = 2000000000ll;

DFM_DEV bool ap_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint32_t* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (clock64() - t0 > AP_WAIT_CLOCKS) {
      *abort_flag = 1;
      atomicOr(err, DFM_DEV_ERR_TIMEOUT);
      return false;
    }
  }
}

// Wait with the time limit alone, whatever the abort flag says (the way out of
// an aborted CTA, whose copies and products are still in flight).
DFM_DEV void mbar_drain(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity) && clock64() - t0 <= AP_WAIT_CLOCKS) {
  }
}

// Barrier `id` over `threads` threads (whole warps); the AND of their predicates.
DFM_DEV bool ap_meet(int id, int threads, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(ok)), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}

template <bool kFp16>
DFM_DEV uint32_t ap_pack(float a, float b) {
  if constexpr (kFp16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16(a, b);
  }
}

// 32 TMEM columns of this thread's lane, asynchronously: x is there after
// ap_landed, whose operands keep the compiler from using it earlier.
DFM_DEV void ap_load(uint32_t taddr, float (&x)[32]) {
  tmem_ld32(taddr, reinterpret_cast<uint32_t(&)[32]>(x));
}
DFM_DEV void ap_landed(float (&x)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]), "+f"(x[6]),
                 "+f"(x[7]), "+f"(x[8]), "+f"(x[9]), "+f"(x[10]), "+f"(x[11]), "+f"(x[12]), "+f"(x[13]),
                 "+f"(x[14]), "+f"(x[15]), "+f"(x[16]), "+f"(x[17]), "+f"(x[18]), "+f"(x[19]), "+f"(x[20]),
                 "+f"(x[21]), "+f"(x[22]), "+f"(x[23]), "+f"(x[24]), "+f"(x[25]), "+f"(x[26]), "+f"(x[27]),
                 "+f"(x[28]), "+f"(x[29]), "+f"(x[30]), "+f"(x[31])
               :
               : "memory");
}

// 0 x + sum for two 16-bit values.
template <bool kFp16>
DFM_DEV uint32_t ap_zero_times(uint32_t x, uint32_t sum) {
  uint32_t r;
  if constexpr (kFp16)
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(sum));
  else
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(sum));
  return r;
}

// Two 16-bit values, an infinity or a NaN replaced by zero.
template <bool kFp16>
DFM_DEV uint32_t ap_finite(uint32_t x) {
  constexpr uint32_t E = kFp16 ? 0x7c007c00u : 0x7f807f80u;
  return x & ~__vcmpeq2(x & E, E);
}

// The lowest n bits, n clamped to [0, 32].
DFM_DEV uint32_t low_bits(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }

// Which of the 32 keys from kc on a row sees: [lo, hi), and drafted tokens of a tree.
DFM_DEV uint32_t ap_sees(int kc, int lo, int hi, int base, unsigned long long bits) {
  uint32_t see = low_bits(hi - kc) & ~low_bits(lo - kc);
  const int o = base - kc;   // drafted token 0's bit in this word
  if (bits) see |= o >= 32 || o <= -64 ? 0u
                 : o >= 0 ? static_cast<uint32_t>(bits << o) : static_cast<uint32_t>(bits >> -o);
  return see;
}

template <bool kFp16>
DFM_DEV float ap_value(uint16_t x) {
  return kFp16 ? __half2float(__ushort_as_half(x)) : __uint_as_float(static_cast<uint32_t>(x) << 16);
}

// A row's special values of V: two bits a dim, an infinity seen (x) or a negative one
// (y), both where their sum is a NaN.
template <int D>
struct ApSpecial {
  uint2 dims[D / 32];
};

// Notes those of the key tile at k0 that the row sees; poison: the tile's keys that have
// any; fresh: the segment's first.
template <int D, bool kFp16>
__device__ __noinline__ void ap_special_note(const ApParams& p, int seq, int kv, int k0, const uint32_t* poison,
                                             int lo, int hi, int base, unsigned long long bits,
                                             ApSpecial<D>* sp, bool fresh) {
  if (fresh) *sp = ApSpecial<D>{};
  for (int c = 0; c < 128; c += 32) {
    for (uint32_t w = poison[c >> 5] & ap_sees(k0 + c, lo, hi, base, bits); w; w &= w - 1) {
      const int key = k0 + c + __ffs(w) - 1, block = p.by_block(key);
      const int cb = p.bt[static_cast<size_t>(seq) * p.max_blocks + block];
      if (cb < 0 || cb >= p.num_blocks) continue;   // (read as zeros)
      const size_t row = static_cast<size_t>(cb) * p.block_size + (key - block * p.block_size);
      const uint16_t* v = static_cast<const uint16_t*>(p.v) + (row * p.KVH + kv) * D;
      for (int d = 0; d < D; ++d) {
        constexpr uint32_t E = kFp16 ? 0x7c00u : 0x7f80u;
        if ((v[d] & E) != E) continue;
        const bool nan = v[d] & (E ^ 0x7fffu), neg = v[d] >> 15;
        if (nan || !neg) sp->dims[d >> 5].x |= 1u << (d & 31);
        if (nan || neg) sp->dims[d >> 5].y |= 1u << (d & 31);
      }
    }
  }
}

// Adds them to dims [lo, hi) of what this thread wrote: the row's output, or its
// partial (out null).
template <int D, bool kFp16>
__device__ __noinline__ void ap_special_put(const ApSpecial<D>* a, const ApSpecial<D>* b, int lo, int hi,
                                            uint16_t* out, float* po) {
  for (int d = lo; d < hi; ++d) {
    const uint32_t bit = 1u << (d & 31);
    const bool inf = ((a ? a->dims[d >> 5].x : 0) | (b ? b->dims[d >> 5].x : 0)) & bit;
    const bool neg = ((a ? a->dims[d >> 5].y : 0) | (b ? b->dims[d >> 5].y : 0)) & bit;
    if (!inf && !neg) continue;
    const float x = inf && neg ? __int_as_float(0x7fffffff) : inf ? INFINITY : -INFINITY;
    if (out) out[d] = static_cast<uint16_t>(ap_pack<kFp16>(ap_value<kFp16>(out[d]) + x, 0.f));
    else po[static_cast<size_t>(d >> 3) * (AP_ROWS * 8) + (d & 7)] += x;
  }
}

DFM_DEV void st_global_v8(void* dst, const uint32_t (&v)[8]) {   // 32-byte aligned
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

DFM_DEV void ld_global_v8(const float* src, float4& a, float4& b) {   // 32-byte aligned
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(a.x), "=f"(a.y), "=f"(a.z), "=f"(a.w), "=f"(b.x), "=f"(b.y), "=f"(b.z), "=f"(b.w)
               : "l"(src));
}

// Two fp32 operations in one instruction.
DFM_DEV uint64_t f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
DFM_DEV void f2_split(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
DFM_DEV uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
DFM_DEV uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
DFM_DEV uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^x of two scores on the fp32 pipe: x = n + f with n the nearest integer, 2^f by
// the polynomial of degree 5 fitted at Chebyshev nodes of [-1/2, 1/2] (1e-7
// relative), times 2^n, which for n = -127 comes out as an exact 0 (masked scores are
// -inf); a NaN stays one.
constexpr float AP_E0 = 1.00000008f, AP_E1 = 0.693147207f, AP_E2 = 0.240221073f, AP_E3 = 0.055503272f, AP_E4 = 0.00967604193f, AP_E5 = 0.00134004369f;
DFM_DEV void ap_exp2_pair(uint64_t x, float& a, float& b) {
  constexpr float kRound = 12582912.f;   // 1.5 * 2^23: adding it rounds to an integer
  f2_split(x, a, b);
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(a), "f"(-127.f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(b), "f"(-127.f));
  const uint64_t y = f2(a, b), t = f2_add(y, f2(kRound, kRound));
  const uint64_t f = f2_add(y, f2_fma(t, f2(-1.f, -1.f), f2(kRound, kRound)));
  uint64_t q = f2(AP_E5, AP_E5);
  q = f2_fma(q, f, f2(AP_E4, AP_E4));
  q = f2_fma(q, f, f2(AP_E3, AP_E3));
  q = f2_fma(q, f, f2(AP_E2, AP_E2));
  q = f2_fma(q, f, f2(AP_E1, AP_E1));
  q = f2_fma(q, f, f2(AP_E0, AP_E0));
  float ta, tb;
  f2_split(t, ta, tb);
  // kRound's low bits are zero: t's hold n, and (n << 23) + the bits of 1 is 2^n
  q = f2_mul(q, f2(__uint_as_float((__float_as_uint(ta) << 23) + 0x3f800000u),
                   __uint_as_float((__float_as_uint(tb) << 23) + 0x3f800000u)));
  f2_split(q, a, b);
}

DFM_DEV float ap_max32(const float (&x)[32], float top) {
  float t0 = top, t1 = x[0];
#pragma unroll
  for (int e = 1; e < 31; e += 2) {
    t0 = fmaxf(t0, x[e]);
    t1 = fmaxf(t1, x[e + 1]);
  }
  return fmaxf(fmaxf(t0, t1), x[31]);
}

// The cap: x = (cap / scale) tanh(S scale / cap) of a raw score S (x scale is the
// capped score).  Below half the cap, tanh y = y q(y^2) with q the cubic fitted at
// Chebyshev nodes of [0, 1/4] (6e-7 relative), its coefficients scaled so that x = S
// q(S^2): 2.5 instructions a score on the fp32 pipe.  From there on 1 - 2 / (1 + e^{2y}),
// 10^-7 caps off: two special-function operations, of which an SM does 16 a clock,
// so that they and the softmax's exponential would take three times the products' time.
// Which of the two counts is a score's own matter in tiles with masks or a bias and
// a row's own in the others, so that no other row, and no key that the row does not
// see, has a say in its result.
constexpr float AP_T0 = 0.999999464f, AP_T1 = -0.33326377f, AP_T2 = 0.131909163f, AP_T3 = -0.0444185946f;
DFM_DEV bool ap_far(float big, const ApParams& p) {   // (a NaN is not above the bound and stays one)
  return big > p.cap_hot;
}
DFM_DEV uint64_t ap_cap_near(uint64_t y, const ApParams& p) {
  const uint64_t z = f2_mul(y, y);
  return f2_mul(y, f2_fma(f2_fma(f2_fma(f2(p.cap_q[2], p.cap_q[2]), z, f2(p.cap_q[1], p.cap_q[1])), z,
                                 f2(p.cap_q[0], p.cap_q[0])), z, f2(AP_T0, AP_T0)));
}
DFM_DEV float ap_cap_far(float x, const ApParams& p) {
  float t;   // (volatile: computed for every row, a branch around it costs more)
  asm volatile("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(1.f + fast_exp2(x * p.cap_in)));
  return fmaf(-2.f * p.cap_b, t, p.cap_b);
}
DFM_DEV void ap_cap(float (&x)[32], const ApParams& p) {   // none of the warp's is past the bound
#pragma unroll
  for (int e = 0; e < 32; e += 2) f2_split(ap_cap_near(f2(x[e], x[e + 1]), p), x[e], x[e + 1]);
}
// Where some of the warp's scores are past the bound: 64 scores in TMEM, capped each
// its way (kRows false), or those of the rows that are `far` alone, with the row's largest
// as the result.  (Calls, so that the kernel's other paths have its registers: inlined
// they spilled, and 16 trees of 33 to 63 tokens with a cap far above their scores
// took 70.9 us instead of 63.5.)
template <bool kRows>
__device__ __noinline__ float ap_cap_some(uint32_t taddr, bool far, const ApParams& p) {
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 64; c += 32) {
    float x[32];
    ap_load(taddr + c, x);
    ap_landed(x);
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      const float fa = ap_cap_far(x[e], p), fb = ap_cap_far(x[e + 1], p);
      if (kRows) {
        x[e] = far ? fa : x[e];
        x[e + 1] = far ? fb : x[e + 1];
      } else {
        float a, b;
        f2_split(ap_cap_near(f2(x[e], x[e + 1]), p), a, b);
        x[e] = ap_far(fabsf(x[e]), p) ? fa : a;
        x[e + 1] = ap_far(fabsf(x[e + 1]), p) ? fb : b;
      }
    }
    if (kRows) top = ap_max32(x, top);
    tmem_st32(taddr + c, reinterpret_cast<uint32_t(&)[32]>(x));
  }
  tmem_wait_st();
  return top;
}
DFM_DEV float ap_cap_one(float x, const ApParams& p) {   // below half the cap
  const float z = x * x;
  return x * fmaf(fmaf(fmaf(p.cap_q[2], z, p.cap_q[1]), z, p.cap_q[0]), z, AP_T0);
}
DFM_DEV float ap_abs32(const float (&x)[32], float big) {
#pragma unroll
  for (int e = 0; e < 32; ++e) big = fmaxf(big, fabsf(x[e]));
  return big;
}

// x += slope e, one instruction a score (e is an immediate; in pairs, with e from
// registers, 6000 packed tokens took 84.6 us instead of 79.8): with the row's and the
// chunk's shifts, the distance bias.
DFM_DEV void ap_slope(float (&x)[32], float slope) {
#pragma unroll
  for (int e = 0; e < 32; ++e) x[e] = fmaf(slope, static_cast<float>(e), x[e]);
}
// x -= slope |d - e|
DFM_DEV void ap_slope_abs(float (&x)[32], float slope, int d) {
  const float d0 = static_cast<float>(d);
#pragma unroll
  for (int e = 0; e < 32; ++e) x[e] = fmaf(-slope, fabsf(d0 - static_cast<float>(e)), x[e]);
}
// -inf where the row does not see the key
DFM_DEV void ap_mask(float (&x)[32], uint32_t see) {
  if (__all_sync(0xffffffffu, see == ~0u)) return;
#pragma unroll
  for (int e = 0; e < 32; ++e) x[e] = (see >> e) & 1 ? x[e] : -INFINITY;
}

// ---------------------------------------------------------------- the kernel
// A cap and a distance bias on the scores have kernels of their own: what only they
// need costs the others registers.
template <int D, bool kCap, bool kBias, bool kFp16>
__global__ void __launch_bounds__(AP_THREADS, 1)
    llm_append_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ ApParams p) {
  using S = ApSmem<D>;
  constexpr bool kMod = kCap || kBias, kLateCap = kCap && !kBias;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem + S::OFF_Q;
  uint8_t* sK = smem + S::OFF_K;
  uint8_t* sV = smem + S::OFF_V;
  float2* sML = reinterpret_cast<float2*>(smem + S::OFF_ML);
  ApNear& near = *reinterpret_cast<ApNear*>(smem + S::OFF_NEAR);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
  uint64_t* k_empty = k_full + S::RING;
  uint64_t* v_full = k_empty + S::RING;
  uint64_t* v_ready = v_full + S::RING;   // V without special values: arrivals of its two warps
  uint64_t* v_empty = v_ready + S::RING;
  uint64_t* s_full = v_empty + S::RING;   // [2] per stream
  uint64_t* p_full = s_full + 2;          // [2][2] its two halves of P: arrivals of its four warps
  uint64_t* o_full = p_full + 4;          // [2]
  uint64_t* q_full = o_full + 2;
  uint64_t* q_empty = q_full + 1;
  uint64_t* drain = q_empty + 1;
  uint32_t* poison = reinterpret_cast<uint32_t*>(drain + 1);   // [S::RING][4]
  uint32_t* tmem_slot = poison + S::RING * 4;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((5 * S::RING + 11) * 8 + S::RING * 16 + 8 <= 512, "barrier area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::RING; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_ready[i], 2);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch(&tm_q);
    tma_prefetch(&tm_k);
    tma_prefetch(&tm_v);
  }
  if (warp == AP_SOFT_WARPS + 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  pdl_wait();
  if (p.near_plan) near.make(p, *reinterpret_cast<ApNear::Seqs*>(sQ));
  ApWalk walk(p, near);
  ApSegment sg;

  if (warp == AP_SOFT_WARPS) {
    // ------------------------------------------------------------ TMA
    const int per_tile = AP_KT / p.box_rows;         // boxes along the keys
    const int box_bytes = p.box_rows * 128;
    int g = 0, nseg = 0;
    bool ok = true;
    while (ok && walk.next(p, sg)) {
      if (sg.i1 == sg.i0) continue;
      const int* bt = p.bt + static_cast<size_t>(sg.f.seq) * p.max_blocks;
      // lane = (box along the keys, 64-dim half); lanes past the tile's boxes are idle
      const int box = lane / S::BOXES, half = lane % S::BOXES;
      // The cache blocks of 32 boxes, those of the tiles from i on, a lane's each: -2 if
      // nobody sees the box.  With 16-row boxes that is 4 tiles' worth; looked up a tile
      // at a time, 64 single tokens over 16-row pages took 126 us instead of 112.
      auto blocks_from = [&](int i) {
        i += lane / per_tile;
        const int key = (sg.top - i) * AP_KT + lane % per_tile * p.box_rows;
        if (i >= sg.i1 || key + p.box_rows <= sg.f.lo || key >= sg.f.hi) return -2;
        const int b = bt[p.by_block(key)];
        return b < 0 ? -1 : b;
      };
      const int ahead = 32 / per_tile;
      int now = blocks_from(sg.i0), next = blocks_from(sg.i0 + ahead), used = 0;
      if (lane == 0) {
        ok = nseg == 0 || ap_wait(q_empty, (nseg - 1) & 1, abort_flag, p.err);
        if (ok) {
          const int nt = sg.narrow ? 1 : 2;
          mbar_arrive_expect_tx(q_full, nt * S::BOXES * p.G * p.RT * 128);
          for (int x = 0; x < nt; ++x)
            for (int b = 0; b < S::BOXES; ++b)
              tma_load_3d(sQ + x * S::TILE + b * S::HALF, &tm_q, q_full, b * 64, sg.kv * p.G,
                          sg.f.row0 + sg.f.t0 + x * p.RT);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      ++nseg;
      for (int i = sg.i0; ok && i < sg.i1; ++i, ++g) {
        const int slot = g % S::RING;
        const int key = (sg.top - i) * AP_KT + box * p.box_rows;
        const int row = key - p.by_block(key) * p.block_size;
        int cb = __shfl_sync(0xffffffffu, now, used * per_tile + box);
        const bool mine = box < per_tile && cb != -2;
        if (++used == ahead) {
          used = 0;
          now = next;
          next = blocks_from(i + 1 + ahead);
        }
        if (mine && (cb < 0 || cb >= p.num_blocks)) {
          if (half == 0) atomicOr(p.err, DFM_DEV_ERR_PAGE);
          cb = p.num_blocks;   // out of range: zeros
        }
        const int bytes = __popc(__ballot_sync(0xffffffffu, mine)) * box_bytes;
        const int dst = slot * S::TILE + half * S::HALF + box * box_bytes;
        if (lane == 0) {
          ok = g < S::RING || ap_wait(&k_empty[slot], ((g / S::RING) & 1) ^ 1, abort_flag, p.err);
          if (ok) mbar_arrive_expect_tx(&k_full[slot], bytes);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        if (mine) tma_load_4d(sK + dst, &tm_k, &k_full[slot], half * 64, sg.kv, row, cb);
        if (lane == 0) {
          ok = g < S::RING || ap_wait(&v_empty[slot], ((g / S::RING) & 1) ^ 1, abort_flag, p.err);
          if (ok) mbar_arrive_expect_tx(&v_full[slot], bytes);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) {
          ++g;
          break;
        }
        if (mine) tma_load_4d(sV + dst, &tm_v, &v_full[slot], half * 64, sg.kv, row, cb);
      }
    }
    if (lane == 0) {
      // Copies must have landed before the CTA's memory is gone, also those that a
      // warp which gave up did not wait for.
      if (nseg > 0) mbar_drain(q_full, (nseg - 1) & 1);
      for (int x = g > S::RING ? g - S::RING : 0; x < g; ++x) {
        mbar_drain(&k_full[x % S::RING], (x / S::RING) & 1);
        mbar_drain(&v_full[x % S::RING], (x / S::RING) & 1);
      }
    }
  } else if (warp == AP_SOFT_WARPS + 1) {
    // ------------------------------------------------------------ MMA
    // The whole warp walks and waits, so that descriptors are built in uniform
    // registers; one elected lane issues.
    {
      const uint32_t fmt = kFp16 ? 0u : (1u << 7) | (1u << 10);
      const uint32_t base = (1u << 4) | fmt | (static_cast<uint32_t>(AP_ROWS >> 4) << 24);
      const uint32_t idesc_s = base | (static_cast<uint32_t>(AP_KT >> 3) << 17);
      const uint32_t idesc_o = base | (static_cast<uint32_t>(D >> 3) << 17) | (1u << 16);
      const bool leader = elect_one();
      const uint64_t dq = umma_desc_sw128(smem_u32(sQ)), dk = umma_desc_sw128(smem_u32(sK)),
                     dv = umma_desc_sw128_mn(smem_u32(sV), S::HALF);
      int g = 0, nseg = 0;
      int np[2] = {0, 0};        // probability tiles taken per stream
      bool ok = true;
      auto commit = [&](uint64_t* bar) {
        if (leader) umma_commit(bar);
      };
      // S_s = Q_x K^T for the K tile of ring position `at`
      auto scores = [&](int s, int x, int at) {
        const uint64_t q = dq + x * (S::TILE >> 4), k = dk + (at % S::RING) * (S::TILE >> 4);
        const uint32_t d = tmem + s * AP_KT;
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            constexpr int H16 = S::HALF >> 4;
            umma_bf16(d, q + (kk >> 2) * H16 + (kk & 3) * 2, k + (kk >> 2) * H16 + (kk & 3) * 2, idesc_s,
                      kk > 0);
          }
          umma_commit(&s_full[s]);
        }
      };
      auto k_wait = [&](int at) {
        ok = ok && ap_wait(&k_full[at % S::RING], (at / S::RING) & 1, abort_flag, p.err);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      };
      // O_s += P_s V, half a key tile at a time
      auto values = [&](int s, int at, bool first) {
        const uint64_t v = dv + (at % S::RING) * (S::TILE >> 4);
        const uint32_t d = tmem + 256 + s * D, a = tmem + s * AP_KT;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          ok = ok && ap_wait(&p_full[2 * s + h], np[s] & 1, abort_flag, p.err) &&
               (h > 0 || ap_wait(&v_ready[at % S::RING], (at / S::RING) & 1, abort_flag, p.err));
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) return;
          tc_fence_after();
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < AP_KT / 32; ++kk)
              umma_f16_ts(d, a + h * 32 + kk * 8, v + (h * (AP_KT / 2) * 128 + kk * 2048) / 16, idesc_o,
                          !first || h > 0 || kk > 0);
          }
        }
        ++np[s];
      };
      while (ok && walk.next(p, sg)) {
        const int nt = sg.i1 - sg.i0;
        if (nt == 0) continue;
        ok = __all_sync(0xffffffffu, ap_wait(q_full, nseg & 1, abort_flag, p.err));
        ++nseg;
        if (sg.narrow) {
          for (int i = 0; i < 2 && i < nt; ++i) {
            k_wait(g + i);
            if (!ok) break;
            scores(i, 0, g + i);
            commit(&k_empty[(g + i) % S::RING]);
            if (i == nt - 1) commit(q_empty);
          }
          for (int i = 0; ok && i < nt; ++i) {
            const int s = i & 1;
            values(s, g + i, i < 2);
            if (!ok) break;
            commit(&v_empty[(g + i) % S::RING]);
            if (i + 2 >= nt) commit(&o_full[s]);
            if (i + 2 < nt) {
              k_wait(g + i + 2);
              if (!ok) break;
              scores(s, 0, g + i + 2);
              commit(&k_empty[(g + i + 2) % S::RING]);
              if (i + 2 == nt - 1) commit(q_empty);
            }
          }
        } else {
          k_wait(g);
          if (!ok) break;
          scores(0, 0, g);
          scores(1, 1, g);
          commit(&k_empty[g % S::RING]);
          if (nt == 1) commit(q_empty);
          for (int i = 0; ok && i < nt; ++i) {
            for (int s = 0; s < 2; ++s) {
              values(s, g + i, i == 0);
              if (!ok) break;
              if (s == 1) commit(&v_empty[(g + i) % S::RING]);
              if (i == nt - 1) {
                commit(&o_full[s]);
                continue;
              }
              if (s == 0) k_wait(g + i + 1);
              if (!ok) break;
              scores(s, s, g + i + 1);
              if (s == 1) {
                commit(&k_empty[(g + i + 1) % S::RING]);
                if (i + 1 == nt - 1) commit(q_empty);
              }
            }
          }
        }
        g += nt;
      }
      commit(drain);   // products in flight read shared memory and TMEM
      if (leader) mbar_drain(drain, 0);
    }
  } else if (warp > AP_SOFT_WARPS) {
    // ------------------------------------------------------------ special rows of V
    const int w = warp - AP_SOFT_WARPS - 2;
    int g = 0;
    bool ok = true;
    while (ok && walk.next(p, sg)) {
      for (int i = sg.i0; i < sg.i1; ++i, ++g) {
        const int slot = g % S::RING;
        ok = __all_sync(0xffffffffu, ap_wait(&v_full[slot], (g / S::RING) & 1, abort_flag, p.err));
        if (!ok) break;
        const int k0 = (sg.top - i) * AP_KT;
        if (k0 < sg.f.fmin || k0 + AP_KT > sg.f.fmax) {
          for (int x = 0; x < 2; ++x) {
            const int r = w * 64 + x * 32 + lane, key = k0 + r;
            uint8_t* row = sV + slot * S::TILE + r * 128;
            const bool seen = key >= sg.f.lo && key < sg.f.hi;
            bool special = false;
            // (where all rows see the key, a special value is all rows' own)
            if (seen && (key < sg.f.fmin || key >= sg.f.fmax)) {
              // 0 x is NaN for an infinity or a NaN, and stays in the sum
              uint32_t sum = 0;
#pragma unroll 4
              for (int c = 0; c < 8 * S::BOXES; ++c) {
                const uint4 u = *reinterpret_cast<const uint4*>(row + (c >> 3) * S::HALF + (((c & 7) ^ (r & 7)) << 4));
                sum = ap_zero_times<kFp16>(u.x, ap_zero_times<kFp16>(u.y, sum));
                sum = ap_zero_times<kFp16>(u.z, ap_zero_times<kFp16>(u.w, sum));
              }
              special = (sum & 0x7fff7fffu) != 0;
            }
            if (!seen) {
#pragma unroll 4
              for (int c = 0; c < 8 * S::BOXES; ++c)
                *reinterpret_cast<uint4*>(row + (c >> 3) * S::HALF + (((c & 7) ^ (r & 7)) << 4)) =
                    make_uint4(0, 0, 0, 0);
            } else if (special) {
#pragma unroll 1
              for (int c = 0; c < 8 * S::BOXES; ++c) {
                uint4& u = *reinterpret_cast<uint4*>(row + (c >> 3) * S::HALF + (((c & 7) ^ (r & 7)) << 4));
                u = make_uint4(ap_finite<kFp16>(u.x), ap_finite<kFp16>(u.y), ap_finite<kFp16>(u.z),
                               ap_finite<kFp16>(u.w));
              }
            }
            const uint32_t word = __ballot_sync(0xffffffffu, special);
            if (lane == 0) poison[slot * 4 + w * 2 + x] = word;
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_ready[slot]);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int s = warp >> 2;                           // stream
    const int r = (warp & 3) * 32 + lane;              // row of the tile, TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + s * AP_KT + lane_off, tO = tmem + 256 + lane_off;
    const int tok_of = p.by_g(r), head_of = r - tok_of * p.G;
    int g = 0, ns = 0;                                 // V tiles of the CTA, score tiles of the stream
    int no[2] = {0, 0};                                // segments each stream had tiles in
    bool ok = true;
    ApCut cut;
    cut.last = -1;
    // this thread's row of the segment
    int j, pos, lo, hi, base;
    bool valid, warp_valid;
    unsigned long long bits;
    float slope;
    auto row = [&]() {
      j = sg.f.t0 + (sg.narrow ? 0 : s * p.RT) + tok_of;
      valid = tok_of < p.RT && j < sg.f.t0 + sg.f.ntok;
      warp_valid = __any_sync(0xffffffffu, valid);
      base = sg.f.base;
      pos = base + j;
      lo = hi = 0;
      bits = 0;
      slope = 0.f;
      if (!valid) return;
      if (!kBias && p.tree) {   // (trees have no distance bias)
        bits = p.tree[sg.f.row0 + j] & (sg.f.m >= 64 ? ~0ull : (1ull << sg.f.m) - 1);
        hi = base;
      } else {
        ap_keys(p, sg.f.row0, j, base, base + sg.f.m, sg.f.pre, lo, hi);
      }
      if (kBias) slope = p.slopes[sg.kv * p.G + head_of] * (1.4426950408889634f / p.scale_log2);   // in units of x
    };
    bool more = walk.next(p, sg);
    if (more) row();
    while (more) {
      const int nt = sg.i1 - sg.i0;
      const bool narrow = sg.narrow;
      auto sees = [&](int kc) { return ap_sees(kc, lo, hi, base, kBias ? 0 : bits); };
      float m = -INFINITY, l = 0.f;
      bool special = false, special_too = false;   // of V: this stream's, the other's (narrow)
      auto special_of = [&](int stream) {
        return reinterpret_cast<ApSpecial<D>*>(p.special) + (blockIdx.x * 2 + stream) * AP_ROWS + r;
      };
      const int step = narrow ? 2 : 1, i_first = narrow ? s : 0;
#pragma unroll 1
      for (int i = i_first; ok && i < nt; i += step, ++ns) {
        ok = __all_sync(0xffffffffu, ap_wait(&s_full[s], ns & 1, abort_flag, p.err));
        if (!ok) break;
        tc_fence_after();
        const int k0 = (sg.top - sg.i0 - i) * AP_KT;
        const bool full = k0 >= sg.f.fmin && k0 + AP_KT <= sg.f.fmax;
        if (warp_valid) {
          // Two passes over the row's 128 scores in TMEM, 32 at a time so that the
          // code stays small: the maximum, then the probabilities.  With masks, a bias or
          // scores near the cap, the changed scores x go back to TMEM in between; in a tile
          // without masks a row far below the cap leaves it to the second pass, as a polynomial.
          // x scale + shift is the score in log2 units (with a bias, chunk c's 32 keys are
          // c grow further on).
          float shift = 0.f, grow = 0.f, top = -INFINITY;
          float xa[32], xb[32];
          auto ld = [&](float (&x)[32], int c) { ap_load(tS + c * 32, x); };
          bool stored = kBias || !full;
          bool raw = false;   // this row leaves its cap to the second pass
          float near_top = 0.f;
          if (!stored) {
            float big = 0.f;
            ld(xa, 0);
#pragma unroll 1
            for (int c = 0; c < 4; c += 2) {
              ap_landed(xa);
              ld(xb, c + 1);
              top = ap_max32(xa, top);
              if (kCap) big = ap_abs32(xa, big);
              ap_landed(xb);
              if (c == 0) ld(xa, 2);
              top = ap_max32(xb, top);
              if (kCap) big = ap_abs32(xb, big);
            }
            if constexpr (kCap) {   // the cap rises with the score: the maximum's is the maximum
              // (16 trees of 33 to 63 tokens with a cap: 63.5 us; 75.4 with the capped scores
              // stored back and read again)
              raw = !ap_far(big, p);
              stored = __any_sync(0xffffffffu, valid && !raw);
              near_top = ap_cap_one(top, p);
              top = -INFINITY;
            }
          }
          if (stored) {
            const bool behind = k0 + AP_KT - 1 <= pos || (p.causal && !p.prefix);
            if (kBias && behind) {
              shift = -slope * p.scale_log2 * static_cast<float>(pos - k0);
              grow = 32.f * slope;
            }
#pragma unroll 1
            for (int c = 0; c < 128; c += 64) {
              const uint32_t sa = full ? ~0u : sees(k0 + c), sb = full ? ~0u : sees(k0 + c + 32);
              const bool masked = __any_sync(0xffffffffu, (sa & sb) != ~0u);
              if (masked && !__any_sync(0xffffffffu, (sa | sb) != 0)) {   // nobody's
#pragma unroll
                for (int e = 0; e < 32; ++e) xa[e] = -INFINITY;
                tmem_st32(tS + c, reinterpret_cast<uint32_t(&)[32]>(xa));
                tmem_st32(tS + c + 32, reinterpret_cast<uint32_t(&)[32]>(xa));
                continue;
              }
              if (kLateCap && full) {
                top = fmaxf(top, ap_cap_some<true>(tS + c, !raw, p));
                continue;
              }
              ap_load(tS + c, xa);
              ap_load(tS + c + 32, xb);
              ap_landed(xa);
              ap_landed(xb);
              if constexpr (kCap) {
                if (__any_sync(0xffffffffu, ap_far(ap_abs32(xa, ap_abs32(xb, 0.f)), p))) {
                  ap_cap_some<false>(tS + c, false, p);
                  ap_load(tS + c, xa);
                  ap_load(tS + c + 32, xb);
                  ap_landed(xa);
                  ap_landed(xb);
                } else {
                  ap_cap(xa, p);
                  ap_cap(xb, p);
                }
              }
              if constexpr (kBias) {
                if (behind) {   // every key the row sees is at or before it: |p - k| = (p - k0) - c
                  ap_slope(xa, slope);
                  ap_slope(xb, slope);
                } else {
                  ap_slope_abs(xa, slope, pos - k0 - c);
                  ap_slope_abs(xb, slope, pos - k0 - c - 32);
                }
              }
              if (masked) {
                ap_mask(xa, sa);
                ap_mask(xb, sb);
              }
              if constexpr (kBias) {
                const float c32 = static_cast<float>(c >> 5);
                top = fmaxf(top, fmaf(grow, c32, ap_max32(xa, -INFINITY)));
                top = fmaxf(top, fmaf(grow, c32 + 1.f, ap_max32(xb, -INFINITY)));
              } else {
                top = ap_max32(xb, ap_max32(xa, top));
              }
              if (kMod || masked) {
                tmem_st32(tS + c, reinterpret_cast<uint32_t(&)[32]>(xa));
                tmem_st32(tS + c + 32, reinterpret_cast<uint32_t(&)[32]>(xb));
              }
            }
            if (!full) {
              // special values of V that this row sees, noted until the product takes V
              const int slot = (g + i) % S::RING;
              ok = __all_sync(0xffffffffu, ap_wait(&v_ready[slot], ((g + i) / S::RING) & 1, abort_flag, p.err));
              if (!ok) break;
              uint32_t bad = 0;
              for (int c = 0; c < 4; ++c) bad |= poison[slot * 4 + c] & sees(k0 + c * 32);
              if (bad) {
                ap_special_note<D, kFp16>(p, sg.f.seq, sg.kv, k0, poison + slot * 4, lo, hi, base,
                                          kBias ? 0 : bits, special_of(s), !special);
                special = true;
              }
            }
            tmem_wait_st();
          }
          if (raw) top = near_top;
          const float mt = fmaf(top, p.scale_log2, shift);
          // Each row raises its maximum by its own scores alone, so that its result does
          // not depend on the rows beside it: of other tokens, and past the unit's last
          // token on the next sequence's queries or, past RT G, on what the shared memory held.
          const bool raise = valid && mt > m + AP_TAU;
          if (i == i_first) {
            m = mt;
          } else if (__any_sync(0xffffffffu, raise)) {
            // the stream's last product is done: this tile's scores came after it
            const float a = raise ? fast_exp2(m - mt) : 1.f;
            l *= a;
            m = raise ? mt : m;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              ap_load(tO + s * D + c, xb);
              ap_landed(xb);
#pragma unroll
              for (int e = 0; e < 32; ++e) xb[e] *= a;
              tmem_st32(tO + s * D + c, reinterpret_cast<uint32_t(&)[32]>(xb));
            }
          }
          const float ms = shift - (m == -INFINITY ? 0.f : m);
          const uint64_t sc = f2(p.scale_log2, p.scale_log2);
          grow *= p.scale_log2;
          uint64_t sum0 = f2(0.f, 0.f), sum1 = f2(0.f, 0.f);
          uint32_t pk[32];
          // kind 1: every score takes the cap's polynomial; 2: those of rows that are raw;
          // 0: none
          auto second_pass = [&](auto kind) {
            constexpr int kLate = decltype(kind)::value;
            uint64_t y0, y1, y2, y3;
            if constexpr (kLate > 0) {
              const bool q = kLate == 1 || raw;
              const float c0 = q ? p.cap_y[0] : p.scale_log2, c1 = q ? p.cap_y[1] : 0.f,
                          c2 = q ? p.cap_y[2] : 0.f, c3 = q ? p.cap_y[3] : 0.f;
              y0 = f2(c0, c0), y1 = f2(c1, c1), y2 = f2(c2, c2), y3 = f2(c3, c3);
            }
            auto probabilities = [&](const float (&x)[32], int at, int c) {
              const float mc = kBias ? fmaf(grow, static_cast<float>(c), ms) : ms;
              const uint64_t sh = f2(mc, mc);
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                float a, b;
                const uint64_t v = f2(x[e], x[e + 1]);
                uint64_t y;
                if constexpr (kLate > 0) {
                  const uint64_t z = f2_mul(v, v);
                  y = f2_fma(v, f2_fma(f2_fma(f2_fma(y3, z, y2), z, y1), z, y0), sh);
                } else {
                  y = f2_fma(v, sc, sh);
                }
                if ((e >> 1) % AP_EXP_OF < AP_EXP_POLY) {
                  ap_exp2_pair(y, a, b);
                } else {
                  f2_split(y, a, b);
                  a = fast_exp2(a);
                  b = fast_exp2(b);
                }
                if (e & 2) sum1 = f2_add(sum1, f2(a, b));
                else sum0 = f2_add(sum0, f2(a, b));
                pk[at + (e >> 1)] = ap_pack<kFp16>(a, b);
              }
            };
            ld(xa, 0);
            // (P's chunks lie on scores that have been read)
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              ap_landed(xa);
              ld(xb, 2 * h + 1);
              probabilities(xa, 0, 2 * h);
              ap_landed(xb);
              if (h == 0) ld(xa, 2);
              probabilities(xb, 16, 2 * h + 1);
              tmem_st32(tS + h * 32, pk);
              tmem_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&p_full[2 * s + h]);
            }
          };
          if (kLateCap && full && !stored) second_pass(std::integral_constant<int, kLateCap ? 1 : 0>{});
          else if (kLateCap && __any_sync(0xffffffffu, valid && raw)) second_pass(std::integral_constant<int, kLateCap ? 2 : 0>{});
          else second_pass(std::integral_constant<int, 0>{});
          float a, b;
          f2_split(f2_add(sum0, sum1), a, b);
          l += a + b;
        } else if (lane == 0) {   // nobody reads this warp's rows
          mbar_arrive(&p_full[2 * s]);
          mbar_arrive(&p_full[2 * s + 1]);
        }
      }
      // ------------------------------------------------ the segment's rows
      const int n0 = narrow ? (nt + 1) / 2 : nt, n1 = narrow ? nt / 2 : nt;
      const bool whole = sg.whole();
      const int slot = blockIdx.x * 2 + (sg.i0 > 0 ? 0 : 1);
      if (sg.i0 == 0 && !whole) {     // the end of the share cuts this unit
        cut.row = sg.f.row0 + sg.f.t0;
        cut.ntok = sg.f.ntok;
        cut.kv = sg.kv;
        cut.last = (sg.kv * walk.line + sg.f.at + sg.f.lead(p.RT) + ((sg.tiles - 1) << !sg.narrow)) / walk.share;
      }
      const size_t row_off = (static_cast<size_t>(sg.f.row0 + j) * p.H + sg.kv * p.G + head_of) * D;
      const bool put = valid, warp_put = warp_valid;
      g += nt;
      more = walk.next(p, sg);
      if (more) row();     // its loads run under what follows
      float w0 = 1.f, w1 = 0.f;       // weights of O_0 and O_1 (narrow)
      if (narrow) {
        sML[s * AP_ROWS + r] = make_float2(m, copysignf(l, special ? -1.f : 1.f));
        ok = ap_meet(1, 32 * AP_SOFT_WARPS, ok);
        float2 o = sML[(1 - s) * AP_ROWS + r];
        special_too = signbit(o.y);
        o.y = fabsf(o.y);
        const float mm = fmaxf(m, o.x);
        const float wm = m == -INFINITY ? 0.f : fast_exp2(m - mm), wo = o.x == -INFINITY ? 0.f : fast_exp2(o.x - mm);
        w0 = s ? wo : wm;
        w1 = s ? wm : wo;
        l = __fadd_rn(__fmul_rn(l, wm), __fmul_rn(o.y, wo));   // the same in both warpgroups
        m = mm;
      }
      if (ok && n0 > 0 && (narrow || s == 0))
        ok = __all_sync(0xffffffffu, ap_wait(&o_full[0], no[0] & 1, abort_flag, p.err));
      if (ok && n1 > 0 && (narrow || s == 1))
        ok = __all_sync(0xffffffffu, ap_wait(&o_full[1], no[1] & 1, abort_flag, p.err));
      no[0] += n0 > 0;
      no[1] += n1 > 0;
      if (ok && warp_put) {
        tc_fence_after();
        // columns of this warpgroup: all of its own tile's, or half of the shared one's
        const int c_lo = narrow ? s * (D / 2) : 0, c_hi = narrow ? c_lo + D / 2 : D;
        const int tile = narrow ? 0 : s;
        const size_t part = (static_cast<size_t>(slot) * 2 + tile) * AP_ROWS;
        float* po = p.part_o + part * D + r * 8;
        uint16_t* out = static_cast<uint16_t*>(p.out) + row_off;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        w0 *= whole ? inv : 1.f;
        w1 *= whole ? inv : 1.f;
        if (!whole && put && (!narrow || s == 0)) p.part_ml[part + r] = make_float2(m, l);
#pragma unroll 1
        for (int c = c_lo; c < c_hi; c += 32) {
          float v[32], o1[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = o1[e] = 0.f;
          if (n0 > 0) ap_load(tO + (narrow ? 0 : s * D) + c, v);
          if (narrow && n1 > 0) ap_load(tO + D + c, o1);
          ap_landed(v);
          ap_landed(o1);
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = fmaf(v[e], w0, o1[e] * w1);
          if (!put) continue;
          // a thread's row, whole 32-byte sectors at a time
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 16) {
              uint32_t pk[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) pk[x] = ap_pack<kFp16>(v[e + 2 * x], v[e + 2 * x + 1]);
              st_global_v8(out + c + e, pk);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              st_global_v8(po + static_cast<size_t>((c + e) >> 3) * (AP_ROWS * 8),
                           reinterpret_cast<const uint32_t(&)[8]>(v[e]));
          }
        }
        if (special || special_too)
          ap_special_put<D, kFp16>(special ? special_of(s) : nullptr, special_too ? special_of(1 - s) : nullptr,
                                   c_lo, c_hi, whole ? out : nullptr, po);
      }
      tc_fence_before();
      if (narrow) ok = ap_meet(1, 32 * AP_SOFT_WARPS, ok);   // both have read O_0 and O_1
    }
    if (threadIdx.x == 0) p.cuts[blockIdx.x] = cut;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == AP_SOFT_WARPS + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- split units
// Joins the units that lie in several shares:
//   out = sum_j 2^(m_j - M) O_j / sum_j 2^(m_j - M) l_j over the shares j.
// An item is 8 dims of 32 rows, which lie next to each other in the partials.  A
// load of another SM's partial takes over a microsecond, so the items of all cuts
// are spread evenly over one wave of blocks (three to an SM with three shares in
// flight a thread: 0.5 to 1 us faster than two with four), and where there are few, 2 or 4
// warps take an item's shares in turn (their sums are added in the warps' order).
template <int D, bool kFp16>
__global__ void __launch_bounds__(AP_COMBINE_THREADS, AP_COMBINE_BLOCKS)
    llm_append_combine_kernel(const ApParams p) {
  constexpr int CB = 3, DG = D / 8, WARPS = AP_COMBINE_THREADS / 32;
  __shared__ float part[WARPS][10][32];
  __shared__ int2 sums[WARPS];
  __shared__ int4 cuts[AP_MAX_CTAS];    // ApCut: row, ntok, kv, last
  __shared__ int starts[AP_MAX_CTAS];
  pdl_trigger();
  pdl_wait();
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  auto row_groups = [&](int tokens) { return (tokens * p.G + 31) >> 5; };
  int n = 0;
  if (t < p.ctas) {
    const int4 c = *reinterpret_cast<const int4*>(&p.cuts[t]);
    if (c.w > t) n = (row_groups(min(c.y, p.RT)) + row_groups(c.y - min(c.y, p.RT))) * DG;
    cuts[t] = c;
  }
  int2 all;
  const int begin = block_scan<WARPS>(make_int2(n, 0), sums, all).x;
  if (t < p.ctas) starts[t] = begin;
  __syncthreads();
  const int items = all.x;
  if (items == 0) return;
  const int room = gridDim.x * WARPS;
  const int team = items * 4 <= room ? 4 : items * 2 <= room ? 2 : 1;   // warps to an item
  const int k = warp % team, at_once = WARPS / team;
  for (int i0 = blockIdx.x * at_once; i0 < items; i0 += gridDim.x * at_once) {
    const int it = min(i0 + warp / team, items - 1);
    int b = 0;                  // the last cut that starts at or before the item
    for (int hi = p.ctas - 1; b < hi;) {
      const int mid = (b + hi + 1) >> 1;
      if (starts[mid] <= it) b = mid; else hi = mid - 1;
    }
    const int4 cut = cuts[b];
    const int row = cut.x, ntok = cut.y, kv = cut.z, last = cut.w;
    const int item = it - starts[b], dg = item % DG, rg = item / DG;
    const int first = min(ntok, p.RT), groups1 = row_groups(first), tile = rg >= groups1;
    const int r = (tile ? rg - groups1 : rg) * 32 + lane;
    const bool mine = i0 + warp / team < items && r < (tile ? ntok - first : first) * p.G;
    float M = -INFINITY, L = 0.f, acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    for (int c0 = b + k; mine && c0 <= last; c0 += CB * team) {
      float2 ml[CB];
      float4 o[CB][2];
#pragma unroll
      for (int x = 0; x < CB; ++x) {
        const int c = c0 + x * team;
        const bool in = c <= last;
        const size_t at = (static_cast<size_t>(c) * 2 + (c > b ? 0 : 1)) * 2 + tile;
        const float* src = p.part_o + at * AP_ROWS * D + (dg * AP_ROWS + r) * 8;
        ml[x] = in ? p.part_ml[at * AP_ROWS + r] : make_float2(-INFINITY, 0.f);
        o[x][0] = o[x][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (in) ld_global_v8(src, o[x][0], o[x][1]);
      }
      float Mn = M;
#pragma unroll
      for (int x = 0; x < CB; ++x) Mn = fmaxf(Mn, ml[x].x);
      const float a = M == -INFINITY ? 0.f : fast_exp2(M - Mn);
      L *= a;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] *= a;
#pragma unroll
      for (int x = 0; x < CB; ++x) {
        const float wt = ml[x].x == -INFINITY ? 0.f : fast_exp2(ml[x].x - Mn);
        L += wt * ml[x].y;
        acc[0] += wt * o[x][0].x;
        acc[1] += wt * o[x][0].y;
        acc[2] += wt * o[x][0].z;
        acc[3] += wt * o[x][0].w;
        acc[4] += wt * o[x][1].x;
        acc[5] += wt * o[x][1].y;
        acc[6] += wt * o[x][1].z;
        acc[7] += wt * o[x][1].w;
      }
      M = Mn;
    }
    if (team > 1) {
      part[warp][8][lane] = M;
      part[warp][9][lane] = L;
#pragma unroll
      for (int e = 0; e < 8; ++e) part[warp][e][lane] = acc[e];
      __syncthreads();
      if (k == 0) {
        float Mn = M;
        for (int x = 1; x < team; ++x) Mn = fmaxf(Mn, part[warp + x][8][lane]);
        const float a = M == -INFINITY ? 0.f : fast_exp2(M - Mn);
        L *= a;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] *= a;
        for (int x = 1; x < team; ++x) {
          const float mx = part[warp + x][8][lane];
          const float wt = mx == -INFINITY ? 0.f : fast_exp2(mx - Mn);
          L += wt * part[warp + x][9][lane];
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] += wt * part[warp + x][e][lane];
        }
      }
      __syncthreads();
    }
    if (!mine || k != 0) continue;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int tok = p.by_g(r), j = tile * p.RT + tok;
    *reinterpret_cast<uint4*>(
        static_cast<uint16_t*>(p.out) +
        (static_cast<size_t>(row + j) * p.H + kv * p.G + r - tok * p.G) * D + dg * 8) =
        make_uint4(ap_pack<kFp16>(acc[0] * inv, acc[1] * inv), ap_pack<kFp16>(acc[2] * inv, acc[3] * inv),
                   ap_pack<kFp16>(acc[4] * inv, acc[5] * inv), ap_pack<kFp16>(acc[6] * inv, acc[7] * inv));
  }
}

}  // namespace dfm
