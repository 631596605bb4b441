/*
 * Rotary positions, a paged key/value cache and the attention that reads it,
 * on MI355X (gfx950): plan + launch C-ABI.
 *
 * A cache is a pool of P pages of page_size tokens each, for k and for v:
 * element (page, token, head, dim) with the given strides and dim contiguous,
 * so that [P][page_size][Hkv][D] and [P][Hkv][page_size][D] both do.  Sequence
 * b's token j lies in page table[b][j / page_size], slot j % page_size; a table
 * entry outside [0, P) holds no page.  kv_len[b] counts b's tokens with the new
 * ones of the present call, of which there are n_b: one for every sequence
 * without cu_q, else cu_q[b + 1] - cu_q[b], rows cu_q[b] .. of the new tokens'
 * tensors.  New token i of b has position kv_len[b] - n_b + i.
 *
 * All arrays are device memory; index arrays are int32.  No launch reads
 * lengths or tables on the host, so all can be captured into a graph and replayed with
 * other contents (a workspace then is the graph's alone, its counters cleared by a node of
 * the graph).  Contents out of range (a page outside [0, P), positions past
 * the table, cu_q past T) are skipped by the kernels, never followed.  A plan
 * is a plain struct that the caller keeps; the launch plans its descriptor
 * again and refuses one that differs.  Errors: return codes and
 * tx_get_last_error() (tx_dot.h).
 */
#ifndef TRITON_EXT_AMD_TX_CACHE_H
#define TRITON_EXT_AMD_TX_CACHE_H

#include "triton_ext/tx_dot.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rotary positions ----------------------------------------------------
 * x [Z][N][H][head_dim] by strides.  With angle a = position * inv_freq[i]
 * (the product and its reduction to one turn in 64 bits), c = scale * cos a and
 * s = scale * sin a, pair i of every head goes to
 *     (x1 c - x2 s, x2 c + x1 s)             inverse: s -> -s
 * where (x1, x2) are dims (i, i + rot_dim / 2), or (2 i, 2 i + 1) when
 * interleaved; dims from rot_dim on are copied.  The inverse is the transposed
 * map: of y's gradient it makes x's.  fp32 arithmetic, rounded once.  out may be
 * x itself. */
typedef struct tx_rotary_desc {
  int64_t Z, N, H;
  int32_t head_dim, rot_dim; /* rot_dim even, 0 < rot_dim <= head_dim */
  int32_t dtype;             /* TX_F32, TX_F16 or TX_BF16 */
  int32_t interleaved, inverse;
  int32_t pos_bits; /* 32 or 64: positions are int32 or int64 */
  float scale;
  int32_t reserved; /* 0 */
  int64_t pos_sz;   /* elements from one batch's positions to the next's (0: shared) */
  /* element strides (batch, token, head); none is filled in.  Those of x may be 0
   * (a broadcast view) */
  int64_t x_sz, x_sn, x_sh;
  int64_t o_sz, o_sn, o_sh;
} tx_rotary_desc;

typedef struct tx_rotary_plan {
  tx_rotary_desc desc;
  double flops, bytes;
  int32_t vec;         /* elements of one access (the launch takes 1 where a base is less aligned) */
  int32_t head_lanes;  /* threads that share a token's heads */
  int32_t grid_x, block_threads;
} tx_rotary_plan;

TX_API int tx_rotary_plan_create(const tx_rotary_desc *desc, tx_rotary_plan *plan);
TX_API int tx_rotary_launch(const tx_rotary_plan *plan, const void *x, const void *positions,
                            const float *inv_freq, void *out, void *stream);

/* ---- new tokens into the cache -------------------------------------------
 * k, v [T][Hkv][head_dim] are written into the pages of their sequences, k (and
 * q [T][Hq][head_dim], into q_out) rotated at the token's position first where
 * rot_dim > 0.  An e4m3 cache takes x / scale[head], saturated at +-448, to nearest
 * even (scales NULL: 1).  Tokens without a page are not written (their q is
 * rotated all the same); rows of q from cu_q[B] on are copied. */
typedef struct tx_paged_append_desc {
  int64_t T, B;
  int64_t pages, table_width; /* of the cache; entries of a table row */
  int32_t Hq, Hkv;            /* Hq 0: no q */
  int32_t head_dim, rot_dim, page_size; /* page_size a power of two */
  int32_t dtype;              /* TX_F16 or TX_BF16: q, k, v, q_out */
  int32_t cache_type;         /* dtype or TX_F8E4M3 */
  int32_t interleaved, ragged; /* ragged: cu_q is given; else T == B */
  float scale;
  int64_t q_st, q_sh, o_st, o_sh; /* element strides (token, head) */
  int64_t k_st, k_sh, v_st, v_sh;
  int64_t kc_sp, kc_st, kc_sh, vc_sp, vc_st, vc_sh; /* caches: (page, token, head) */
  int64_t table_s;            /* elements from one table row to the next */
} tx_paged_append_desc;

typedef struct tx_paged_append_plan {
  tx_paged_append_desc desc;
  double flops, bytes;
  int32_t vec, head_lanes, grid_x, block_threads;
} tx_paged_append_plan;

TX_API int tx_paged_append_plan_create(const tx_paged_append_desc *desc, tx_paged_append_plan *plan);
TX_API int tx_paged_append_launch(const tx_paged_append_plan *plan, const void *q, const void *k,
                                  const void *v, void *q_out, void *k_cache, void *v_cache,
                                  const int32_t *page_table, const int32_t *kv_len,
                                  const int32_t *cu_q, const float *inv_freq, const float *k_scale,
                                  const float *v_scale, void *stream);

/* ---- attention of new tokens over the cache ------------------------------
 * Of new token i of sequence b at position p, query head h and kv head h / (Hq / Hkv):
 *     o = sum_j e^(sm_scale q.k_j) v_j / sum_j e^(sm_scale q.k_j)
 * over its tokens j < kv_len[b] that have a page, j <= p if causal, and j > p - window
 * if window > 0.  lse [T][Hq] (fp32, optional): log2 of the sum of e^(..).  A token
 * that attends to nothing, and rows from cu_q[B] on, get o = 0 and lse = -inf.  e4m3
 * caches: k and v times k_scale[kv head], v_scale[kv head] (fp32; NULL: 1).  What
 * the cache holds where nothing is attended to may be anything, NaN included, outside
 * [0, kv_len) and in pages the table does not name.  Products on the matrix cores
 * with fp32 sums, softmax in fp32; p (relative to a maximum of the row's keys up to there, and up to
 * 2^8) is rounded to q's type before p . v.  A sequence has at most 2^31 - 128 tokens.  The
 * order of sums depends on the lengths alone: the same call gives the same bits. */
typedef struct tx_paged_attn_desc {
  int64_t T, B;
  int64_t pages, table_width;
  int32_t Hq, Hkv, head_dim, page_size; /* head_dim a multiple of 8 (e4m3 cache: 16), <= 256 */
  int32_t dtype;      /* q, o: TX_F16 or TX_BF16 */
  int32_t cache_type; /* dtype or TX_F8E4M3 */
  int32_t causal, window, ragged;
  float sm_scale;     /* >= 0 */
  int64_t q_st, q_sh, o_st, o_sh; /* element strides, multiples of 16 bytes */
  int64_t k_sp, k_st, k_sh, v_sp, v_st, v_sh;
  int64_t table_s;
} tx_paged_attn_desc;

typedef struct tx_paged_attn_plan {
  tx_paged_attn_desc desc;
  int32_t variant; /* the kernel: 0, 1: waves share out the keys, 2: the rows */
  int32_t rows;    /* query rows (token x head of one kv head) of a unit of work: 16, 32, 128 */
  int32_t slots;   /* workspace places for parts of a unit's keys */
  int32_t units;   /* workgroups, which share all units' keys in equal runs */
  int32_t grid_x, block_threads;
  int64_t workspace_bytes; /* as tx_dot_launch's workspace: zeroed before its first use, never
                            * shared by launches that may overlap */
} tx_paged_attn_plan;

TX_API int tx_paged_attn_plan_create(const tx_paged_attn_desc *desc, tx_paged_attn_plan *plan);
TX_API int tx_paged_attn_launch(const tx_paged_attn_plan *plan, const void *q, const void *k_cache,
                                const void *v_cache, const int32_t *page_table,
                                const int32_t *kv_len, const int32_t *cu_q, const float *k_scale,
                                const float *v_scale, void *o, float *lse, void *workspace,
                                size_t workspace_bytes, void *stream);

/* ---- pages ---------------------------------------------------------------
 * The books of a pool: page_table [S][W], kv_len [S], refs [P], packed int32; refs[p]
 * counts the table entries that hold page p, 0 = free.  A sequence of n tokens uses
 * its first ceil(n / page_size) entries.  Every call reads one set of books and writes another,
 * which may be the same arrays.  Free pages are taken in ascending order. */
#define TX_PAGE_CACHES 128
typedef struct tx_page_desc {
  int64_t S, W, P;
  int64_t n;         /* page_fork: children; page_copy: pages */
  int32_t page_size; /* a power of two */
  int32_t caches;    /* tensors that hold pages, at most TX_PAGE_CACHES */
  /* bytes from one page to the next and of one page, of each tensor: multiples of 16 */
  int64_t stride[TX_PAGE_CACHES], bytes[TX_PAGE_CACHES];
} tx_page_desc;

/* Checks desc, and gives the bytes of scratch memory that each of the calls below needs for
 * it (any contents, 8-byte aligned). */
TX_API int tx_page_workspace(const tx_page_desc *desc, int64_t *bytes);

/* Page src[i] of every cache is copied to page dst[i], i < n.  Entries outside
 * [0, P) are skipped.  No dst may be another dst or a src (but its own). */
TX_API int tx_page_copy(const tx_page_desc *desc, void *const *caches, const int32_t *src,
                        const int32_t *dst, void *stream);
/* kv_len goes up to new_len (never down, and to W * page_size at most), with free pages
 * for what that adds, in the order of sequences.  *missing: the pages that there
 * were too few (those entries get -1). */
TX_API int tx_page_reserve(const tx_page_desc *desc, const int32_t *page_table,
                           const int32_t *kv_len, const int32_t *refs, const int32_t *new_len,
                           int32_t *table_out, int32_t *len_out, int32_t *refs_out,
                           int32_t *missing, void *workspace, void *stream);
/* Row child[i] becomes a sequence that shares the pages of parent[i], but for a last page
 * that is not full, which is copied to a free one.  Children are empty rows, each named
 * once and no parent; pairs with an index outside [0, S) are skipped. */
TX_API int tx_page_fork(const tx_page_desc *desc, void *const *caches, const int32_t *page_table,
                        const int32_t *kv_len, const int32_t *refs, const int32_t *parent,
                        const int32_t *child, int32_t *table_out, int32_t *len_out,
                        int32_t *refs_out, int32_t *missing, void *workspace, void *stream);
/* Sequences with drop[s] != 0 (bytes) give their pages back and become empty. */
TX_API int tx_page_free(const tx_page_desc *desc, const int32_t *page_table, const int32_t *kv_len,
                        const int32_t *refs, const uint8_t *drop, int32_t *table_out,
                        int32_t *len_out, int32_t *refs_out, void *stream);
/* With U pages in use: the used pages from U on, in order, move to the free pages
 * below U, in order, in the caches and in the books.  *moved: how many. */
TX_API int tx_page_compact(const tx_page_desc *desc, void *const *caches,
                           const int32_t *page_table, const int32_t *refs, int32_t *table_out,
                           int32_t *refs_out, int32_t *moved, void *workspace, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* TRITON_EXT_AMD_TX_CACHE_H */
