/*
 * fa2_ops.h - C ABI of the operators around the attention entry points of
 * fa2.h: query / key norms with the position rotation, and the paged K/V cache
 * held in 4 bits (writer, reader, decode and speculative decode attention).
 *
 * No counterpart in the reference (harsh-vsingh/triton-kernels), whose kernels
 * take finished queries and keys and 16/32-bit caches; the paged layout
 * (block tables, lengths, prefix sums) and the decode semantics are those of
 * its kernels/decode.py and kernels/speculative_decode.py.
 *
 * As in fa2.h: all pointers but the parameter blocks are device pointers;
 * strides are in elements, the last dimension is contiguous and rows start on
 * 16-byte boundaries; status codes are enum fa2_status; errors are reported
 * before any launch; no allocation, no host synchronisation.
 */
#ifndef FA2_OPS_H_
#define FA2_OPS_H_

#include "fa2.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- norms of queries and keys, with the rotation ---------------------------
 *
 * For each head row x (head_dim values) of q and k:
 *   y = x * rsqrt(mean(x^2) + eps) * weight
 * and the first rotary_dim values of y, in pairs (a, b), become
 *   (a cos - b sin, b cos + a sin),
 * with cos and sin of pair i of the row's token in rope[position][i] and
 * rope[position][rotary_dim / 2 + i].  Pairs are (i, i + rotary_dim / 2), or
 * with `interleaved` (2 i, 2 i + 1).  Computed in fp32, rounded once: a bf16 or fp32
 * row whose sum of squares passes fp32's range gives zeros.  A token whose
 * position is outside [0, positions) gives NaN rows.
 *
 * Token t of q is row t % q_rows of batch t / q_rows: token-major [T, H, D] has
 * q_rows = T (q_sb unused), [B, H, M, D] has q_rows = M; likewise k. */
typedef struct fa2_norm_rope_params {
  int32_t dtype;        /* enum fa2_dtype of q, k and the outputs             */
  int32_t weight_dtype; /* `dtype`, or FA2_DTYPE_F32                          */
  int32_t interleaved;
  float eps;            /* >= 0                                               */
  int64_t tokens, q_heads, kv_heads;
  int64_t head_dim;     /* 16, 32, 64, 128 or 256                             */
  int64_t rotary_dim;   /* 0 .. head_dim, a multiple of 16                    */
  int64_t positions;    /* rows of rope                                       */
  int64_t rope_stride;  /* elements, a multiple of 4                          */
  int64_t q_rows, k_rows;
  int64_t q_sb, q_sh, q_ss, k_sb, k_sh, k_ss;     /* (batch, head, row)       */
  int64_t qo_sb, qo_sh, qo_ss, ko_sb, ko_sh, ko_ss;
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  const void* q_weight; /* [head_dim]                                         */
  const void* k_weight;
  const float* rope;    /* [positions, rotary_dim]: cosines, then sines       */
  const void* position; /* [tokens], int32 (int64 with position_64)           */
  int32_t position_64;
  int32_t reserved0;
} fa2_norm_rope_params;

int fa2_norm_rope(const fa2_norm_rope_params* p, void* stream);

/* ---- the paged cache in 4 bits ------------------------------------------------
 *
 * codes  uint8 [num_pages, kv_heads, page_size, head_dim / 2]
 * scales uint8 [num_pages, kv_heads, page_size, head_dim / 32]
 * both contiguous, the scales from a 4-byte boundary; head_dim 64, 128 or 256; a
 * page's codes less than 2^30 bytes.  Value d of a row is nibble d % 2 (0: low) of byte
 * d / 2, an E2M1 number (sign, two exponent bits, one mantissa bit: 0 .5 1 1.5 2 3 4
 * 6), times 2^(scale - 127) of its block d / 32; scale 255 is NaN.  (OCP MX FP4
 * with blocks of 32.)  Logical row n of sequence b is row n % page_size of page
 * table[b][n / page_size].
 *
 * The writer gives a block the least power of two at which its largest value is
 * at most 6 after rounding, kept between 2^-23 and 2^13 for fp16 rows and 2^-100
 * and 2^125 for the others (so that every cached value is exact in the rows'
 * type), rounds to nearest, ties to even, and saturates.  A block that holds an
 * infinity or NaN is NaN. */
typedef struct fa2_fp4_rows_params {
  int32_t dtype;            /* enum fa2_dtype of the rows                       */
  int32_t reserved0;
  int64_t batch, kv_heads, head_dim;
  int64_t num_rows;         /* rows of k / v                                    */
  int64_t page_size, num_pages;
  int64_t table_width;      /* columns of the block tables (0: they may be NULL) */
  int64_t k_table_stride, v_table_stride;
  int64_t k_ts, k_hs, v_ts, v_hs; /* element strides (row, head) of k / v       */
  void* k;                  /* [num_rows, kv_heads, head_dim]                   */
  void* v;                  /* the four V pointers may all be NULL: K only      */
  uint8_t* k_codes;
  uint8_t* k_scales;
  uint8_t* v_codes;
  uint8_t* v_scales;
  const int32_t* indptr;    /* [batch + 1] prefix sums over the rows            */
  const int32_t* start_pos; /* [batch] first logical position, or NULL (0)      */
  const int32_t* k_block_table;
  const int32_t* v_block_table;
} fa2_fp4_rows_params;

/* Write the rows into the caches (k and v are read).  Rows without a place (a
 * page past the table, a table entry outside the pool) are skipped; two rows of
 * a call must not share one. */
int fa2_fp4_append(const fa2_fp4_rows_params* p, void* stream);

/* Read rows out of the caches (k and v are written).  Rows without a place are
 * zeros; rows outside [indptr[0], indptr[batch]) are left as they are. */
int fa2_fp4_gather(const fa2_fp4_rows_params* p, void* stream);

/* Decode / speculative decode attention over the cache: fa2_decode_fwd's
 * computation (packed heads, bottom-right causal drafts, NaN for a row without
 * keys) on the cache's values, with fp16/bf16 q and o [B, Hq, q_len, D].  The
 * softmax weights enter the P.V product as two 16-bit parts.  Lengths past
 * table_width * page_size count as that; table entries are clamped into the pool. */
typedef struct fa2_fp4_decode_params {
  int32_t dtype;            /* FA2_DTYPE_F16 or FA2_DTYPE_BF16                  */
  int32_t mask;             /* FA2_MASK_NONE or FA2_MASK_CAUSAL_BOTTOM_RIGHT    */
  int64_t batch, q_heads, kv_heads, head_dim, q_len;
  int64_t page_size, num_pages, table_width;
  int64_t k_table_stride, v_table_stride;
  int64_t q_sb, q_sh, q_ss; /* as fa2_decode_fwd: q_sh == q_len * q_ss          */
  int64_t o_sb, o_sh, o_ss;
  const void* q;
  void* o;
  const uint8_t* k_codes;
  const uint8_t* k_scales;
  const uint8_t* v_codes;
  const uint8_t* v_scales;
  const int32_t* kv_lens;       /* [batch]                                      */
  const int32_t* k_block_table; /* [batch, table_width]; NULL where that is 0    */
  const int32_t* v_block_table;
  float softmax_scale;          /* > 0, finite                                  */
  int32_t reserved0;
  void* workspace;          /* 16-byte aligned, any prior content; one per call in flight */
  size_t workspace_bytes;
} fa2_fp4_decode_params;

int fa2_fp4_decode_workspace_size(const fa2_fp4_decode_params* p, size_t* bytes);
int fa2_fp4_decode(const fa2_fp4_decode_params* p, void* stream);

/* sizeof of parameter block `which` (0 norm_rope, 1 fp4_rows, 2 fp4_decode) as
 * compiled into the library; 0 for another number. */
size_t fa2_ops_params_size(int which);

#ifdef __cplusplus
}
#endif

#endif /* FA2_OPS_H_ */
