// Host side of the rotary and append-attention C ABI (include/dllm.h).
// Compiled inside dfm_api.cu's translation unit, after llm_api.cu, whose helpers
// it uses.
#include "llm_append.cuh"
#include "llm_rotary.cuh"

namespace {

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// ---------------------------------------------------------------- rotary
template <typename T, bool INTER>
cudaError_t launch_rotary(RotaryParams& p, cudaStream_t s) {
  constexpr int VP = 16 / sizeof(T);
  const long long heads = p.heads + (p.slots ? 2 * p.kv_heads : 0);
  auto strides_ok = [](std::initializer_list<long long> v) {
    for (long long x : v)
      if (x % VP) return false;
    return true;
  };
  bool vec = p.D % (2 * VP) == 0 && (p.rot / 2) % VP == 0 && p.rot / 2 <= RO_MAX_PAIRS && aligned16(p.q) && aligned16(p.q_out) &&
             strides_ok({p.q_ts, p.q_hs, p.o_ts, p.o_hs});
  if (p.slots)
    vec = vec && aligned16(p.k) && aligned16(p.v) && aligned16(p.k_cache) && aligned16(p.v_cache) &&
          strides_ok({p.k_ts, p.k_hs, p.v_ts, p.v_hs});
  auto blocks = [](long long threads) { return (threads + RO_THREADS - 1) / RO_THREADS; };
  if (!vec) {
    const long long nb = blocks(p.tokens * heads * ((p.D + 1) / 2));
    if (nb > 0x7fffffffll) return cudaErrorInvalidValue;
    return launch_pdl(llm_rotary_scalar_kernel<T, INTER>, dim3(static_cast<unsigned>(nb)),
                      dim3(RO_THREADS), 0, s, p);
  }
  // four tokens to a block where that still leaves every SM a few blocks
  const long long lanes = p.D / (2 * VP);
  const int tb = p.tokens >= 16 * sm_count() ? 4 : 1;
  if (heads * lanes * tb > 0x7fffffffll) return cudaErrorInvalidValue;
  p.by_token.set(static_cast<int>(heads * lanes));
  p.by_lanes.set(static_cast<int>(lanes));
  p.by_pairs.set(p.rot / 2);
  return launch_pdl(tb == 4 ? llm_rotary_kernel<T, INTER, 4> : llm_rotary_kernel<T, INTER, 1>,
                    dim3(static_cast<unsigned>((p.tokens + tb - 1) / tb)), dim3(RO_THREADS), 0, s, p);
}

// ---------------------------------------------------------------- append attention
struct ApWs {
  size_t head, units, ubase, start, cuts, special, part_ml, part_o, total;
};

int ap_max_units(int tokens, int n, int RT) {
  const long long u = (static_cast<long long>(tokens) + 2 * RT - 1) / (2 * RT) + n;
  return u > 0x7fffffff ? 0 : static_cast<int>(u);
}

ApWs ap_ws(int tokens, int n, int G, int D, int ctas) {
  auto up = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
  ApWs w;
  w.head = 256;   // after the error word
  w.units = w.head + 256;
  w.ubase = w.units + up(sizeof(ApUnit) * static_cast<size_t>(ap_max_units(tokens, n, AP_ROWS / G)));
  w.start = w.ubase + up(4 * (static_cast<size_t>(n) + 1));
  w.cuts = w.start + up(4 * (static_cast<size_t>(ctas) + 1));
  w.special = w.cuts + up(sizeof(ApCut) * static_cast<size_t>(ctas));
  w.part_ml = w.special + up(static_cast<size_t>(ctas) * 2 * AP_ROWS * D / 4);   // two bits a dim
  w.part_o = w.part_ml + up(static_cast<size_t>(ctas) * 4 * AP_ROWS * sizeof(float2));
  w.total = w.part_o + static_cast<size_t>(ctas) * 4 * AP_ROWS * D * 4;
  return w;
}

// CTAs of the append kernel: one to an SM.
int ap_ctas() { return sm_count() < AP_MAX_CTAS ? sm_count() : AP_MAX_CTAS; }

bool ap_shape_ok(int tokens, int n, int H, int KVH, int D) {
  return tokens >= 0 && n >= 1 && H >= 1 && KVH >= 1 && H % KVH == 0 && H / KVH <= AP_ROWS &&
         (D == 64 || D == 128) && ap_max_units(tokens, n, AP_ROWS / (H / KVH)) > 0;
}

// A paged cache as [num_blocks][block_size][kv_heads][D]: boxes of 64 dims x
// `rows` positions of one block.
bool map_ap_cache(CUtensorMap* m, const DllmAppend& a, const void* base, int rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t D = a.head_dim, KVH = a.num_kv_heads, bs = a.block_size;
  cuuint64_t dims[4] = {D, KVH, bs, static_cast<cuuint64_t>(a.num_blocks)};
  cuuint64_t strides[3] = {D * 2, KVH * D * 2, bs * KVH * D * 2};
  cuuint32_t box[4] = {64, 1, static_cast<cuuint32_t>(rows), 1};
  cuuint32_t es[4] = {1, 1, 1, 1};
  return fn(m, a.dtype == DLLM_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            4, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The queries as [tokens][H][D]: a box is the G heads of one kv head of RT tokens.
bool map_ap_q(CUtensorMap* m, const DllmAppend& a, int G, int RT) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(a.num_heads),
                        static_cast<cuuint64_t>(a.tokens)};
  // (a dimension of one element has any stride: it is not stepped over)
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.num_heads > 1 ? a.q_head_stride : a.head_dim) * 2,
                           static_cast<cuuint64_t>(a.tokens > 1 ? a.q_token_stride : a.head_dim) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(G), static_cast<cuuint32_t>(RT)};
  cuuint32_t es[3] = {1, 1, 1};
  return fn(m, a.dtype == DLLM_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            3, const_cast<void*>(a.q), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool kCap, bool kBias, bool kFp16>
cudaError_t launch_append(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                          const ApParams& p, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  constexpr int smem = ApSmem<D>::BYTES;
  auto fn = llm_append_kernel<D, kCap, kBias, kFp16>;
  cudaError_t r = smem_attr_once(done, fn, smem);
  if (r != cudaSuccess) return r;
  if (!p.near_plan) {
    r = launch_pdl(llm_append_plan_kernel, dim3(1), dim3(AP_PLAN_THREADS), 0, s, p);
    if (r != cudaSuccess) return r;
  }
  r = launch_pdl(fn, dim3(p.ctas), dim3(AP_THREADS), smem, s, q, k, v, p);
  if (r != cudaSuccess || p.ctas < 2) return r;
  return launch_pdl(llm_append_combine_kernel<D, kFp16>, dim3(p.ctas * AP_COMBINE_BLOCKS),
                    dim3(AP_COMBINE_THREADS), 0, s, p);
}

template <int D, bool kFp16>
cudaError_t launch_append(bool cap, bool bias, const CUtensorMap& q, const CUtensorMap& k,
                          const CUtensorMap& v, const ApParams& p, cudaStream_t s) {
  if (cap)
    return bias ? launch_append<D, true, true, kFp16>(q, k, v, p, s)
                : launch_append<D, true, false, kFp16>(q, k, v, p, s);
  return bias ? launch_append<D, false, true, kFp16>(q, k, v, p, s)
              : launch_append<D, false, false, kFp16>(q, k, v, p, s);
}

}  // namespace

extern "C" {

int dllm_rotary(const DllmRotary* a, void* stream) {
  if (!a) return DFM_ERR_INVALID_ARG;
  if (a->dtype < DLLM_BF16 || a->dtype > DLLM_FP32) return DFM_ERR_UNSUPPORTED;
  if (a->tokens < 0 || a->q_heads < 1 || a->head_dim < 2 || a->head_dim % 2 || a->rot_dim < 2 ||
      a->rot_dim % 2 || a->rot_dim > a->head_dim)
    return DFM_ERR_INVALID_ARG;
  if (!a->turns || !a->positions || !a->q || !a->q_out) return DFM_ERR_INVALID_ARG;
  if (a->k && (!a->v || !a->k_cache || !a->v_cache || !a->slot_mapping || !a->err_word ||
               a->kv_heads < 1 || a->num_slots < 1))
    return DFM_ERR_INVALID_ARG;
  if (a->tokens == 0) return DFM_OK;
  RotaryParams p{};
  p.turns = reinterpret_cast<const unsigned long long*>(a->turns);
  p.positions = a->positions;
  p.q = a->q;
  p.q_out = a->q_out;
  p.q_ts = a->q_token_stride;
  p.q_hs = a->q_head_stride;
  p.o_ts = a->out_token_stride;
  p.o_hs = a->out_head_stride;
  if (a->q == a->q_out && (p.q_ts != p.o_ts || p.q_hs != p.o_hs)) return DFM_ERR_INVALID_ARG;
  if (a->k) {
    p.k = a->k;
    p.v = a->v;
    p.k_cache = a->k_cache;
    p.v_cache = a->v_cache;
    p.slots = a->slot_mapping;
    p.k_ts = a->k_token_stride;
    p.k_hs = a->k_head_stride;
    p.v_ts = a->v_token_stride;
    p.v_hs = a->v_head_stride;
    p.kv_heads = a->kv_heads;
    p.num_slots = a->num_slots;
  }
  p.err = a->err_word;
  p.tokens = a->tokens;
  p.heads = a->q_heads;
  p.D = a->head_dim;
  p.rot = a->rot_dim;
  p.factor = a->factor;
  p.copy_tail = a->q != a->q_out;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool in = a->interleaved != 0;
  cudaError_t r = cudaErrorInvalidValue;
  switch (a->dtype) {
    case DLLM_BF16: r = in ? launch_rotary<__nv_bfloat16, true>(p, s) : launch_rotary<__nv_bfloat16, false>(p, s); break;
    case DLLM_FP16: r = in ? launch_rotary<__half, true>(p, s) : launch_rotary<__half, false>(p, s); break;
    case DLLM_FP32: r = in ? launch_rotary<float, true>(p, s) : launch_rotary<float, false>(p, s); break;
  }
  return r == cudaSuccess ? DFM_OK : DFM_ERR_CUDA;
}

size_t dllm_append_workspace_size(int32_t tokens, int32_t n, int32_t num_heads,
                                  int32_t num_kv_heads, int32_t head_dim) {
  if (!ap_shape_ok(tokens, n, num_heads, num_kv_heads, head_dim)) return 0;
  return ap_ws(tokens, n, num_heads / num_kv_heads, head_dim, ap_ctas()).total;
}

int dllm_append_attention(const DllmAppend* a, void* workspace, size_t workspace_bytes,
                          void* stream) {
  if (!a || !workspace) return DFM_ERR_INVALID_ARG;
  if (a->dtype != DLLM_BF16 && a->dtype != DLLM_FP16) return DFM_ERR_UNSUPPORTED;
  if (!ap_shape_ok(a->tokens, a->n, a->num_heads, a->num_kv_heads, a->head_dim))
    return DFM_ERR_UNSUPPORTED;
  if (!a->q || !a->k_cache || !a->v_cache || !a->cu_seqlens_q || !a->context_lens ||
      !a->block_table || !a->out)
    return DFM_ERR_INVALID_ARG;
  if (a->num_blocks < 1 || a->max_blocks < 1) return DFM_ERR_INVALID_ARG;
  if (a->block_size < 16 || a->block_size % 16) return DFM_ERR_UNSUPPORTED;
  // positions are 32-bit, with room for a tile past the last one
  if (static_cast<long long>(a->max_blocks) * a->block_size > 0x7fffff00ll) return DFM_ERR_UNSUPPORTED;
  if (!(a->scale > 0.f) || !(a->softcap >= 0.f) || !(a->scale < INFINITY) || !(a->softcap < INFINITY) ||
      a->window < 0)
    return DFM_ERR_INVALID_ARG;
  // (beyond these bounds the cap's constants, or the square of a score below it, leave fp32)
  if (a->softcap > 0.f && !(a->scale / a->softcap < 1e37f && a->scale / a->softcap > 1e-18f))
    return DFM_ERR_UNSUPPORTED;
  if (a->tree_masks && (a->prefix_lens || a->first_keys || a->slopes || a->window))
    return DFM_ERR_UNSUPPORTED;
  if (!aligned16(a->q) || !aligned16(a->k_cache) || !aligned16(a->v_cache) || reinterpret_cast<uintptr_t>(a->out) % 32 ||
      (a->tokens > 1 && (a->q_token_stride % 8 || a->q_token_stride < a->head_dim)) ||
      (a->num_heads > 1 && (a->q_head_stride % 8 || a->q_head_stride < a->head_dim)))
    return DFM_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(workspace) % 256) return DFM_ERR_INVALID_ARG;
  const int G = a->num_heads / a->num_kv_heads, RT = AP_ROWS / G, ctas = ap_ctas();
  const ApWs w = ap_ws(a->tokens, a->n, G, a->head_dim, ctas);
  if (workspace_bytes < w.total) return DFM_ERR_WORKSPACE;
  if (a->tokens == 0) return DFM_OK;
  // places in the line of key tiles are 32-bit
  const long long tiles = static_cast<long long>(a->max_blocks) * a->block_size / AP_KT + 2 + AP_WIDE_COST;
  if (2 * tiles * ap_max_units(a->tokens, a->n, RT) > 0x3fffffffll / a->num_kv_heads)
    return DFM_ERR_UNSUPPORTED;
  int rows = AP_KT;
  while (a->block_size % rows) rows /= 2;
  CUtensorMap mq, mk, mv;
  if (!map_ap_q(&mq, *a, G, RT) || !map_ap_cache(&mk, *a, a->k_cache, rows) ||
      !map_ap_cache(&mv, *a, a->v_cache, rows))
    return DFM_ERR_CUDA;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  ApParams p{};
  p.cu = a->cu_seqlens_q;
  p.ctx = a->context_lens;
  p.bt = a->block_table;
  p.prefix = a->prefix_lens;
  p.first = a->first_keys;
  p.tree = reinterpret_cast<const unsigned long long*>(a->tree_masks);
  p.slopes = a->slopes;
  p.v = a->v_cache;
  p.out = a->out;
  p.err = reinterpret_cast<uint32_t*>(ws);
  p.head = reinterpret_cast<ApHead*>(ws + w.head);
  p.units = reinterpret_cast<ApUnit*>(ws + w.units);
  p.ubase = reinterpret_cast<int*>(ws + w.ubase);
  p.start = reinterpret_cast<int*>(ws + w.start);
  p.cuts = reinterpret_cast<ApCut*>(ws + w.cuts);
  p.special = ws + w.special;
  p.part_ml = reinterpret_cast<float2*>(ws + w.part_ml);
  p.part_o = reinterpret_cast<float*>(ws + w.part_o);
  p.tokens = a->tokens;
  p.n = a->n;
  p.H = a->num_heads;
  p.KVH = a->num_kv_heads;
  p.G = G;
  p.RT = RT;
  p.max_units = ap_max_units(a->tokens, a->n, RT);
  p.ctas = ctas;
  // each CTA plans by itself where that fits its shared memory
  p.near_plan = a->n <= AP_NEAR_SEQS && p.max_units <= (a->first_keys ? AP_NEAR_FIRST : AP_NEAR_UNITS);
  p.num_blocks = a->num_blocks;
  p.block_size = a->block_size;
  p.max_blocks = a->max_blocks;
  p.box_rows = rows;
  p.by_g.set(G);
  p.by_unit.set(2 * RT);
  p.by_ctas.set(ctas);
  p.by_block.set(a->block_size);
  p.causal = a->causal != 0;
  p.window = a->window;
  const float log2e = 1.4426950408889634f;
  p.scale_log2 = a->scale * log2e;
  if (a->softcap > 0.f) {
    p.cap_a = a->scale / a->softcap;
    p.cap_b = a->softcap / a->scale;
    p.cap_in = 2.f * log2e * p.cap_a;
    // The powers of a cap_a above 10^6 would overflow: no polynomial.  Those of one below
    // 10^-6 vanish, up to 0.0075 of a score near half the cap: the polynomial only where
    // they do not count (0.02^4 of the score), and above it 1 - 2 / (1 + e^2y), whose
    // error of 10^-7 caps is then 5e-6 of the score.
    p.cap_hot = (p.cap_a > 1e6f ? -1.f : p.cap_a < 1e-6f ? 0.02f : 0.5f) / p.cap_a;
    const float z = p.cap_a * p.cap_a;
    p.cap_q[0] = AP_T1 * z;
    p.cap_q[1] = AP_T2 * z * z;
    p.cap_q[2] = AP_T3 * z * z * z;
    p.cap_y[0] = AP_T0 * p.scale_log2;
    for (int i = 0; i < 3; ++i) p.cap_y[i + 1] = p.cap_q[i] * p.scale_log2;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool cap = a->softcap > 0.f, bias = a->slopes != nullptr, fp16 = a->dtype == DLLM_FP16;
  const cudaError_t r =
      a->head_dim == 128
          ? (fp16 ? launch_append<128, true>(cap, bias, mq, mk, mv, p, s)
                  : launch_append<128, false>(cap, bias, mq, mk, mv, p, s))
          : (fp16 ? launch_append<64, true>(cap, bias, mq, mk, mv, p, s)
                  : launch_append<64, false>(cap, bias, mq, mk, mv, p, s));
  return r == cudaSuccess ? DFM_OK : DFM_ERR_CUDA;
}

}  // extern "C"
