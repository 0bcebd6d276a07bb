/*
 * dllm.h -- C ABI of the B200-native (sm_100a) paged decode attention of the
 * dots.tts LLM backbone (Qwen2: GQA, 12 query heads over 2 kv heads,
 * head_dim 128, paged K/V cache of 256-position blocks).
 *
 * Replaces the decode branch of the reference's Attention layer
 * (nanovllm_dots/layers/attention.py:60-97): the Triton store_kvcache
 * (attention.py:10-47) followed by flash-attn's flash_attn_with_kvcache(q,
 * k_cache, v_cache, cache_seqlens=context_lens, block_table=block_tables,
 * softmax_scale, causal=True) (flash-attn 2.8.3, attention.py:88-97), as driven
 * one token per sequence by BatchedPagedLLM._decode_batch
 * (nanovllm_dots/models/dots/batched_llm.py:177-236).
 *
 * Same library (libdfm.so), status codes and device error bits as dfm.h.
 * Every pointer is a DEVICE pointer; the caller owns every buffer.
 */
#ifndef DLLM_H_
#define DLLM_H_

#include <stddef.h>
#include <stdint.h>

#include "dfm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Workspace bytes of dllm_decode_attention for these bounds (zero-fill it
 * once; it holds the device error word and the split-key partials). */
size_t dllm_decode_workspace_size(int32_t n, int32_t num_heads, int32_t head_dim,
                                  int32_t max_blocks, int32_t block_size);

/* One decode step of one attention layer for n sequences.
 *   q            bf16 [n, num_heads, head_dim]      (after rotary)
 *   k, v         bf16 [n, num_kv_heads, head_dim]   this step's token; NULL with
 *                slot_mapping NULL skips the store
 *   k_cache, v_cache  bf16 [num_blocks, block_size, num_kv_heads, head_dim]
 *   slot_mapping int32 [n]: block * block_size + offset of the token, -1 = no store
 *   context_lens int32 [n]: cached positions the query sees, the token included
 *   block_table  int32 [n, max_blocks]
 *   out          bf16 [n, num_heads, head_dim]
 * head_dim 64 or 128; num_heads a multiple of num_kv_heads with at most 8
 * query heads per kv head; block_size a multiple of 64.  Stream ordered, no
 * allocation, no host synchronisation.  An out-of-range block id or slot, or
 * a context_len outside [1, max_blocks * block_size], sets a device error bit
 * (dllm_read_error) and reads zeros / writes nothing for it. */
int dllm_decode_attention(const void* q, const void* k, const void* v, void* k_cache,
                          void* v_cache, const int32_t* slot_mapping, const int32_t* context_lens,
                          const int32_t* block_table, int32_t n, int32_t num_heads,
                          int32_t num_kv_heads, int32_t head_dim, int32_t num_blocks,
                          int32_t block_size, int32_t max_blocks, float softmax_scale, void* out,
                          void* workspace, size_t workspace_bytes, void* stream);

/* Read and clear the device error word of a workspace; synchronises `stream`.
 * Calls on other streams are seen if the caller has waited for them. */
int dllm_read_error(void* workspace, void* stream, uint32_t* err_word);

/* ---------------------------------------------------------------------------
 * The whole backbone decode step: QwenLLM.forward over one new token per
 * sequence (nanovllm_dots/models/dots/model_llm.py:113-171, as
 * BatchedPagedLLM._decode_batch drives it, batched_llm.py:177-236):
 * per layer RMSNorm -> QKV (+bias) -> rotary -> store + paged attention ->
 * o_proj -> residual -> RMSNorm -> gate|up -> SiLU * up -> down -> residual,
 * then the final RMSNorm.  The residual stream is kept in fp32.
 * ------------------------------------------------------------------------- */

/* Model shape (the Qwen2 config fields) and batch / cache bounds.  hidden a
 * multiple of 512 (1024, 1536 or 2048 in this build); head_dim 128; 2*inter a
 * multiple of 256. */
typedef struct DllmConfig {
  int32_t layers, hidden, heads, kv_heads, head_dim, inter;
  float rms_eps;
  int32_t block_size;   /* cache positions per block (a multiple of 64) */
  int32_t max_blocks;   /* block-table width */
  int32_t max_batch;    /* most sequences per step */
} DllmConfig;

/* Weights, stacked over layers (bf16 [out, in] matrices, fp32 vectors); the
 * layouts of the reference's packed projections (QKVParallelLinear q|k|v,
 * MergedColumnParallelLinear gate|up). */
typedef struct DllmWeights {
  const float* in_norm;     /* [layers][hidden] input_layernorm.weight */
  const void* qkv_w;        /* [layers][(heads + 2 kv_heads) head_dim][hidden] */
  const float* qkv_b;       /* [layers][(heads + 2 kv_heads) head_dim] */
  const void* o_w;          /* [layers][hidden][heads head_dim] (no bias) */
  const float* post_norm;   /* [layers][hidden] post_attention_layernorm.weight */
  const void* gate_up_w;    /* [layers][2 inter][hidden] (no bias) */
  const void* down_w;       /* [layers][hidden][inter] (no bias) */
  const float* final_norm;  /* [hidden] */
  const float* inv_freq;    /* [head_dim / 2] rotary base^(-2i / head_dim) */
} DllmWeights;

/* One step.  k_caches / v_caches are HOST arrays of `layers` device pointers
 * (one cache pair per layer, [num_blocks, block_size, kv_heads, head_dim] bf16);
 * the other pointers are device pointers. */
typedef struct DllmStep {
  int32_t n;
  const void* embeds;             /* bf16 [n, hidden] this step's input embeddings */
  const int32_t* positions;       /* [n] the token's position (its rotary angle) */
  const int32_t* slot_mapping;    /* [n] cache slot of the token */
  const int32_t* context_lens;    /* [n] positions attended, the token included */
  const int32_t* block_table;     /* [n, max_blocks] */
  void* const* k_caches;
  void* const* v_caches;
  int32_t num_blocks;
  void* out;                      /* bf16 [n, hidden] final hidden states */
} DllmStep;

int dllm_create(const DllmConfig* config, const DllmWeights* weights, void** handle);
size_t dllm_step_workspace_size(void* handle);
/* Stream ordered, no allocation, no host synchronisation; the first call with
 * a given workspace or set of caches encodes their TMA descriptors (host work,
 * so make it before stream capture). */
int dllm_decode_step(void* handle, const DllmStep* step, void* workspace, size_t workspace_bytes,
                     void* stream);
int dllm_destroy(void* handle);

/* ---------------------------------------------------------------------------
 * Rotary positions of query and key heads, with the store of k and v into the
 * paged caches (the rotary of nanovllm_dots/layers/rotary_embedding.py:6-47 and
 * store_kvcache, layers/attention.py:10-47, for both pair layouts, part of a
 * head and scaled frequencies).
 * ------------------------------------------------------------------------- */
enum { DLLM_BF16 = 0, DLLM_FP16 = 1, DLLM_FP32 = 2 };

/* Strides are in elements; the last dimension is contiguous. */
typedef struct DllmRotary {
  int32_t dtype;                /* of q, q_out, k, v and the caches (DLLM_*) */
  int32_t tokens;
  int32_t q_heads, kv_heads;    /* kv_heads is not read without the store */
  int32_t head_dim, rot_dim;    /* both even; dims [rot_dim, head_dim) are not turned */
  int32_t interleaved;          /* pairs (2i, 2i + 1), else (i, i + rot_dim / 2) */
  float factor;                 /* on cos and sin (attention factor; 1 for none) */
  const uint64_t* turns;        /* [rot_dim / 2] turns a position, as a binary fraction of 2^64 */
  const int32_t* positions;     /* [tokens] */
  const void* q;                /* [tokens, q_heads, head_dim] */
  void* q_out;                  /* the same shape; may be q with q's strides, else no overlap with
                                 * anything; the caches overlap no other tensor either */
  const void* k;                /* [tokens, kv_heads, head_dim]; NULL skips the store */
  const void* v;
  void* k_cache;                /* [num_slots, kv_heads, head_dim] */
  void* v_cache;
  const int32_t* slot_mapping;  /* [tokens]; -1: not stored */
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  int64_t k_token_stride, k_head_stride, v_token_stride, v_head_stride;
  int64_t num_slots;
  uint32_t* err_word;           /* device word that gets the error bits (a slot past the cache) */
} DllmRotary;

/* Stream ordered, one launch, no allocation, no host synchronisation. */
int dllm_rotary(const DllmRotary* args, void* stream);

/* ---------------------------------------------------------------------------
 * Append attention: the m_i = cu_seqlens_q[i + 1] - cu_seqlens_q[i] newest
 * tokens of each sequence (their K/V is in the cache) over its context_lens[i]
 * cached positions.  Token j of sequence i stands at position
 * context_lens[i] - m_i + j = p and sees the keys k with
 *     k <= p (causal), or k < prefix_lens[i];        every k without causal
 *     k > p - window (window > 0);   k >= first_keys[token]
 * all below context_lens[i].  With tree_masks (m_i <= 64) it sees the history
 * k < context_lens[i] - m_i and the new tokens t whose bit t is set in its
 * mask, whatever their order; the other masks and slopes are not used then.
 * Scores are s = scale q.k, softcap tanh(s / softcap) if softcap > 0, minus
 * slopes[h] |p - k| if slopes; the output is softmax(s) v, and zeros for a
 * token that sees no key.  Scores, softmax and sums are fp32; each softmax
 * weight is rounded to dtype before it meets its row of V (half a step), the
 * result once more.  An infinity or NaN in a K row reaches the tokens that see
 * it, one in a V row its own dims of theirs (as an infinity or NaN), and no
 * other; keys that no token sees are not read beyond the pages of those that
 * are.  Rows of q and out past cu_seqlens_q[n] are not touched.
 * ------------------------------------------------------------------------- */
typedef struct DllmAppend {
  int32_t dtype;                /* of q, caches and out: DLLM_BF16 or DLLM_FP16 */
  int32_t tokens;               /* rows of q and out */
  int32_t n;                    /* sequences */
  int32_t num_heads, num_kv_heads, head_dim;   /* at most 128 query heads a kv head; 64 or 128 */
  int32_t num_blocks, block_size, max_blocks;  /* block_size a multiple of 16 */
  int32_t causal, window;
  float scale, softcap;
  const void* q;                /* [tokens, num_heads, head_dim], 16-byte aligned rows */
  int64_t q_token_stride, q_head_stride;       /* elements, multiples of 8, head_dim or more */
  const void* k_cache;          /* [num_blocks, block_size, num_kv_heads, head_dim] */
  const void* v_cache;
  const int32_t* cu_seqlens_q;  /* [n + 1] */
  const int32_t* context_lens;  /* [n] */
  const int32_t* block_table;   /* [n, max_blocks] */
  const int32_t* prefix_lens;   /* [n] or NULL */
  const int32_t* first_keys;    /* [tokens] or NULL */
  const uint64_t* tree_masks;   /* [tokens] or NULL */
  const float* slopes;          /* [num_heads] or NULL */
  void* out;                    /* [tokens, num_heads, head_dim], 32-byte aligned; may be a
                                 * q of the same strides, else no overlap with anything */
} DllmAppend;

/* Workspace bytes for up to these bounds, 0 if the shape is not supported.
 * Zero-fill the first 256 bytes once (the device error word); nothing else is
 * kept from one call to the next.  Calls that may run at the same time need
 * workspaces of their own. */
size_t dllm_append_workspace_size(int32_t tokens, int32_t n, int32_t num_heads,
                                  int32_t num_kv_heads, int32_t head_dim);

/* Stream ordered, no allocation, no host synchronisation; the launches depend
 * on the arguments but not on the lengths in device memory.  Block tables of
 * nearly 2^31 positions, or of more key tiles in all than 30 bits count, and a
 * softcap below 1e-37 scale or above 1e18 scale are refused
 * (DFM_ERR_UNSUPPORTED).  Lengths that make no sense, a block id out of range
 * or a tree of more than 64 tokens set a device error bit (dllm_read_error);
 * such a sequence's rows are zeros, or untouched where cu_seqlens_q itself is
 * wrong, and such a block reads as zeros. */
int dllm_append_attention(const DllmAppend* args, void* workspace, size_t workspace_bytes,
                          void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DLLM_H_ */
