/*
 * A paged key/value cache held in 4 bits, on MI355X (gfx950): tokens quantised as they are
 * written, the attention over what it holds, and any paged cache read back.  Plan + launch
 * C-ABI; pages, tables, lengths, cu_q and errors as in tx_cache.h.
 *
 * Element (page, token, head, dim) is an e2m1 code (+-{0, .5, 1, 1.5, 2, 3, 4, 6}), two to a
 * byte, the even dim in the low four bits: a head's row is head_dim / 2 bytes, contiguous.
 * Block scales are bytes at (page, token, head, block) by any strides:
 *   TX_SCALE_MX32   e8m0 of 32 dims: value = code * 2^(byte - 127), 255 is NaN
 *   TX_SCALE_NV16   e4m3 of 16 dims: value = code * scale
 * and k_scale, v_scale (fp32 [Hkv], NULL: 1) multiply all of a head.  A cache takes 128 + 8
 * bits of 32 dims (MX32) or 128 + 16 (NV16) where 16-bit caches take 512.
 */
#ifndef TRITON_EXT_AMD_TX_CACHE4_H
#define TRITON_EXT_AMD_TX_CACHE4_H

#include "triton_ext/tx_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct tx_block_scales {
  int32_t mode;     /* TX_SCALE_MX32 or TX_SCALE_NV16 */
  int32_t reserved; /* 0 */
  /* bytes from one (page, token, head, block) to the next, none negative */
  int64_t k_sp, k_st, k_sh, k_sb, v_sp, v_st, v_sh, v_sb;
} tx_block_scales;

/* ---- new tokens into the cache -------------------------------------------
 * As tx_paged_append, but k (after its rotation: sines rounded once to fp32, then two products and their
 * sum) and v are quantised.  Of the block y = x /
 * k_scale[head] with the largest magnitude a:
 *   MX32  e = the least integer with a <= 7 * 2^e, within [-125, 125] (bf16 tokens) or
 *         [-23, 13] (fp16); the scale is e + 127, a code the nearest to y / 2^e
 *   NV16  the scale is a / 6 in e4m3, to nearest even, within [2^-9, 448]; a code the nearest
 *         to y / scale.  Blocks with a below 0.1 have scales among e4m3's subnormals, whose few
 *         bits cost up to a third of a value: k_scale below 1 lifts them
 * Codes go to nearest, ties to the even one, saturated at 6, with y's sign.  A block with a NaN
 * or an infinity gets a scale of NaN and codes of 0.
 * c.cache_type is TX_F4E2M1; c.head_dim a multiple of 32; the caches' strides count bytes and are
 * multiples of 16, as their addresses. */
typedef struct tx_paged_append4_desc {
  tx_paged_append_desc c;
  tx_block_scales s; /* no two scales may share a byte */
} tx_paged_append4_desc;

typedef struct tx_paged_append4_plan {
  tx_paged_append4_desc desc;
  double flops, bytes;
  int32_t whole; /* tokens are read 16 bytes at a time (the launch: where addresses allow it) */
  int32_t run;   /* how a thread has a head's dims: 0: 8 of them, 1: 8 of each half, 2: 8 in pairs */
  int32_t head_lanes, grid_x, block_threads, reserved;
} tx_paged_append4_plan;

TX_API int tx_paged_append4_plan_create(const tx_paged_append4_desc *desc,
                                        tx_paged_append4_plan *plan);
TX_API int tx_paged_append4_launch(const tx_paged_append4_plan *plan, const void *q, const void *k,
                                   const void *v, void *q_out, void *k_cache, void *v_cache,
                                   void *k_block_scale, void *v_block_scale,
                                   const int32_t *page_table, const int32_t *kv_len,
                                   const int32_t *cu_q, const float *inv_freq, const float *k_scale,
                                   const float *v_scale, void *stream);

/* ---- tokens out of a cache -----------------------------------------------
 * Row cu_q[b] + i of k and v [T][Hkv][head_dim] becomes token kv_len[b] - n_b + i of sequence
 * b: what the cache holds times the scales, in fp32, rounded once to out_type.  Rows of
 * tokens without a page, and rows of no sequence, become 0.  cache_type: TX_F16, TX_BF16,
 * TX_F8E4M3 (strides in elements, no block scales) or TX_F4E2M1 (bytes, as above). */
typedef struct tx_paged_read_desc {
  int64_t T, B;
  int64_t pages, table_width;
  int32_t Hkv, head_dim, page_size;
  int32_t cache_type, out_type; /* out_type: TX_F32, TX_F16 or TX_BF16 */
  int32_t ragged;
  int64_t kc_sp, kc_st, kc_sh, vc_sp, vc_st, vc_sh;
  int64_t k_st, k_sh, v_st, v_sh; /* of the rows written, in elements */
  int64_t table_s;
  tx_block_scales s; /* all 0 where cache_type is not TX_F4E2M1 */
} tx_paged_read_desc;

typedef struct tx_paged_read_plan {
  tx_paged_read_desc desc;
  double bytes;
  int32_t vec, head_lanes, grid_x, block_threads; /* vec: 8 or 1 dims of one access */
} tx_paged_read_plan;

TX_API int tx_paged_read_plan_create(const tx_paged_read_desc *desc, tx_paged_read_plan *plan);
TX_API int tx_paged_read_launch(const tx_paged_read_plan *plan, const void *k_cache,
                                const void *v_cache, const void *k_block_scale,
                                const void *v_block_scale, const int32_t *page_table,
                                const int32_t *kv_len, const int32_t *cu_q, const float *k_scale,
                                const float *v_scale, void *k, void *v, void *stream);

/* ---- attention of new tokens over the cache ------------------------------
 * As tx_paged_attn over the values that the cache holds, which are taken in q's type (MX32:
 * exact but for what fp16 has no place for; NV16: exact, in fp16).  p is rounded to bf16 under
 * MX32 with q in bf16, else to fp16, where a weight is off by 2^-32 of the row's sum or by its
 * relative half step, whichever is more.  A row that attends to a
 * token with a scale of NaN, or an MX32 scale above 2^125 (q in fp16: 2^13), in any block of its
 * k or v is NaN as a whole; other rows are not touched by it.  c.cache_type is TX_F4E2M1,
 * c.head_dim a multiple of 32 up to 256; the caches' strides count bytes. */
typedef struct tx_paged_attn4_desc {
  tx_paged_attn_desc c;
  tx_block_scales s;
} tx_paged_attn4_desc;

typedef struct tx_paged_attn4_plan {
  tx_paged_attn4_desc desc;
  int32_t variant; /* the kernel: 0, 1: waves share out the keys, 2: the rows */
  int32_t rows;    /* query rows (token x head of one kv head) of a unit of work */
  int32_t slots, units, grid_x, block_threads; /* as tx_paged_attn_plan's */
  int64_t workspace_bytes;
} tx_paged_attn4_plan;

TX_API int tx_paged_attn4_plan_create(const tx_paged_attn4_desc *desc, tx_paged_attn4_plan *plan);
TX_API int tx_paged_attn4_launch(const tx_paged_attn4_plan *plan, const void *q,
                                 const void *k_cache, const void *v_cache,
                                 const void *k_block_scale, const void *v_block_scale,
                                 const int32_t *page_table, const int32_t *kv_len,
                                 const int32_t *cu_q, const float *k_scale, const float *v_scale,
                                 void *o, float *lse, void *workspace, size_t workspace_bytes,
                                 void *stream);

#ifdef __cplusplus
}
#endif

#endif /* TRITON_EXT_AMD_TX_CACHE4_H */
