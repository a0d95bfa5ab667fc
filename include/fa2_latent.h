/*
 * fa2_latent.h - C ABI of latent attention (keys and values from one shared
 * latent vector a token: cache writer, absorbed and expanded forms) and of
 * attention for trees of drafts.
 *
 * No counterpart in the reference (harsh-vsingh/triton-kernels); the paged
 * layout (block tables, lengths, prefix sums) and the decode semantics are
 * those of its kernels/decode.py and kernels/speculative_decode.py.
 *
 * As in fa2.h: all pointers but the parameter blocks are device pointers;
 * strides are in elements, the last dimension is contiguous and rows start on
 * 16-byte boundaries; status codes are enum fa2_status; errors are reported
 * before any launch; no allocation, no host synchronisation.  Workspaces: 16-byte
 * aligned, any prior content, one per call in flight.
 */
#ifndef FA2_LATENT_H_
#define FA2_LATENT_H_

#include "fa2.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A latent cache: [num_pages, page_size, latent_dim + rope_dim], contiguous, fp16
 * or bf16.  Logical row n of sequence b is row n % page_size of page
 * table[b][n / page_size].  latent_dim 256 or 512, rope_dim 64. */

/* ---- the writer -----------------------------------------------------------------
 *
 * Row x = (c, r) becomes (c * rsqrt(mean(c^2) + eps) * weight, r rotated), with cos
 * and sin of pair i of position n = start_pos[b] + j (the row's logical position) in
 * rope[n][i] and rope[n][rope_dim / 2 + i].  Pairs are (i, i + rope_dim / 2), or with
 * `interleaved` (2 i, 2 i + 1).  Computed in fp32, rounded once.  A position outside
 * [0, positions) gives a NaN row.  Rows without a place in the cache (a page past the
 * table, a table entry outside the pool) are not written there; two rows of a call
 * must not share one.  rows_out (may be NULL) takes every row of a sequence, contiguous;
 * rows outside [indptr[0], indptr[batch]) are left as they are. */
typedef struct fa2_latent_append_params {
  int32_t dtype;        /* FA2_DTYPE_F16 or FA2_DTYPE_BF16                    */
  int32_t weight_dtype; /* `dtype`, or FA2_DTYPE_F32                          */
  int32_t interleaved;
  float eps;            /* >= 0                                               */
  int64_t batch, num_rows, latent_dim, rope_dim;
  int64_t page_size, num_pages, table_width, table_stride;
  int64_t positions;    /* rows of rope                                       */
  int64_t rope_stride;  /* elements, a multiple of 4                          */
  int64_t x_ts;         /* row stride of x                                    */
  const void* x;        /* [num_rows, latent_dim + rope_dim]                  */
  void* rows_out;
  void* cache;
  const void* weight;   /* [latent_dim]                                       */
  const float* rope;    /* [positions, rope_dim]: cosines, then sines         */
  const int32_t* indptr;      /* [batch + 1] prefix sums over the rows        */
  const int32_t* start_pos;   /* [batch] first logical position, or NULL (0)  */
  const int32_t* block_table; /* [batch, table_width]; NULL where that is 0   */
} fa2_latent_append_params;

int fa2_latent_append(const fa2_latent_append_params* p, void* stream);

/* Masks of the decode calls, beside FA2_MASK_NONE and FA2_MASK_CAUSAL_BOTTOM_RIGHT:
 * draft m sees the keys before the drafts (the sequence's last q_len keys) and the
 * drafts d with tree[b][m][d] != 0; q_len at most FA2_TREE_MAX. */
#define FA2_MASK_TREE 3
#define FA2_TREE_MAX 64

/* ---- the absorbed form -------------------------------------------------------------
 *
 * For token m of head h of sequence b: o = sum_n p_n c_n over the sequence's cached
 * rows x_n = (c_n, r_n), p = softmax_n(softmax_scale * q . x_n).  Every head reads the
 * same rows.  Lengths past table_width * page_size count as that; table entries are
 * clamped into the pool; a row without keys is NaN. */
typedef struct fa2_latent_decode_params {
  int32_t dtype;            /* FA2_DTYPE_F16 or FA2_DTYPE_BF16                 */
  int32_t mask;             /* FA2_MASK_NONE, _CAUSAL_BOTTOM_RIGHT or _TREE    */
  int64_t batch, q_heads, q_len, latent_dim, rope_dim;
  int64_t page_size, num_pages, table_width, table_stride;
  int64_t q_sb, q_sh, q_ss; /* q: [batch, q_heads, q_len, latent + rope]       */
  int64_t o_sb, o_sh, o_ss; /* o: [batch, q_heads, q_len, latent]; o_sh == q_len * o_ss */
  int64_t tree_sb, tree_sr; /* bytes; (batch, draft)                           */
  const void* q;
  void* o;
  const void* cache;
  const int32_t* kv_lens;     /* [batch]                                       */
  const int32_t* block_table; /* [batch, table_width]; NULL where that is 0    */
  const uint8_t* tree;        /* FA2_MASK_TREE: [batch, q_len, q_len]          */
  float softmax_scale;        /* > 0, finite                                   */
  int32_t reserved0;
  void* workspace;
  size_t workspace_bytes;
} fa2_latent_decode_params;

int fa2_latent_decode_workspace_size(const fa2_latent_decode_params* p, size_t* bytes);
int fa2_latent_decode(const fa2_latent_decode_params* p, void* stream);

/* ---- the expanded form ---------------------------------------------------------------
 *
 * Prefill: head h's keys are (k[n][h], kr[n]), kr shared by all heads, its values
 * v[n][h]; o[m][h] = sum_n p_n v[n][h], p = softmax_n(softmax_scale * q[m][h] . key_n) under
 * fa2_fwd's masks.  The values have as many dims as k.  Dense: q [batch, heads, q_len,
 * head_dim + rope_dim], k, v and o [batch, heads, len, head_dim], kr [batch, kv_len,
 * rope_dim].  Ragged: [rows, heads, dims] and [rows, rope_dim] with prefix sums.  A row that
 * sees no key is NaN.  Values that a mask hides may be multiplied by zero, so they have to be
 * finite (what lies behind a sequence's end need not be), in the decode calls too. */
typedef struct fa2_latent_prefill_params {
  int32_t layout;           /* FA2_LAYOUT_DENSE or FA2_LAYOUT_RAGGED           */
  int32_t dtype;            /* FA2_DTYPE_F16 or FA2_DTYPE_BF16                 */
  int32_t mask;             /* enum fa2_mask                                   */
  int32_t reserved0;
  int64_t batch, heads;
  int64_t head_dim;         /* of k, v and o: 64 or 128                        */
  int64_t rope_dim;         /* 64                                              */
  int64_t q_len, kv_len;    /* ragged: rows of q and of k                      */
  int64_t q_sb, q_sh, q_ss; /* (batch, head, row); ragged: (unused, head, row) */
  int64_t k_sb, k_sh, k_ss;
  int64_t v_sb, v_sh, v_ss;
  int64_t o_sb, o_sh, o_ss;
  int64_t kr_sb, kr_ss;     /* (batch, row)                                    */
  const void* q;
  const void* k;
  const void* kr;
  const void* v;
  void* o;
  const int32_t* q_indptr;  /* ragged: [batch + 1]                             */
  const int32_t* kv_indptr;
  float softmax_scale;      /* > 0, finite                                     */
  int32_t reserved1;
  void* workspace;
  size_t workspace_bytes;
} fa2_latent_prefill_params;

int fa2_latent_prefill_workspace_size(const fa2_latent_prefill_params* p, size_t* bytes);
int fa2_latent_prefill(const fa2_latent_prefill_params* p, void* stream);

/* ---- trees of drafts over 16-bit K/V caches ------------------------------------------
 *
 * fa2_decode_fwd's computation (its layouts, strides and lengths) with the tree mask,
 * q_len 1 .. FA2_TREE_MAX, fp16 / bf16, head_dim 64, 128 or 256. */
typedef struct fa2_tree_decode_params {
  int32_t layout;           /* enum fa2_layout                                 */
  int32_t dtype;            /* FA2_DTYPE_F16 or FA2_DTYPE_BF16                 */
  int64_t batch, q_heads, kv_heads, head_dim, q_len;
  int64_t kv_len;           /* dense: keys; ragged: total rows; paged: rows of the caches */
  int64_t q_sb, q_sh, q_ss;
  int64_t k_sb, k_sh, k_ss; /* ragged and paged: (unused, head, row)           */
  int64_t v_sb, v_sh, v_ss;
  int64_t o_sb, o_sh, o_ss; /* o_sh == q_len * o_ss                            */
  int64_t page_size, table_width, k_table_stride, v_table_stride;
  int64_t tree_sb, tree_sr; /* bytes; (batch, draft)                           */
  const void* q;
  const void* k;
  const void* v;
  void* o;
  const int32_t* kv_indptr; /* ragged: [batch + 1] prefix sums; paged: [batch] lengths */
  const int32_t* k_block_table;
  const int32_t* v_block_table;
  const uint8_t* tree;      /* [batch, q_len, q_len]                           */
  float softmax_scale;      /* > 0, finite                                     */
  int32_t reserved0;
  void* workspace;
  size_t workspace_bytes;
} fa2_tree_decode_params;

int fa2_tree_decode_workspace_size(const fa2_tree_decode_params* p, size_t* bytes);
int fa2_tree_decode(const fa2_tree_decode_params* p, void* stream);

/* sizeof of parameter block `which` (0 append, 1 latent decode, 2 tree decode, 3 prefill)
 * as compiled into the library; 0 for another number. */
size_t fa2_latent_params_size(int which);

#ifdef __cplusplus
}
#endif

#endif /* FA2_LATENT_H_ */
