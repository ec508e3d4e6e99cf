/*
 * pla_b200 — C ABI of the full-attention operators of a serving step: block tables and slot maps, rotary positions
 * with the per-head norm of queries and keys, and the attention of one new token over a paged cache. They stand
 * beside the linear-attention entries of pla_b200.h (hybrid stacks alternate the two kinds of layer) and follow its
 * conventions: plain argument structures, a stream handle, negative return codes with pla_b200_last_error(),
 * PLA_B200_DEV_* bits OR-ed into `*status` (or into the library's own word) for what only the device can see.
 */
#ifndef PLA_B200_ATTENTION_H_
#define PLA_B200_ATTENTION_H_

#include "pla_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- device status bits of these operators (PLA_B200_DEV_BAD_INTERVAL and _BAD_SLOT are used as well) ---- */
#define PLA_B200_DEV_NO_BLOCK 32    /* the free list ran out: the pages and slots concerned are -1 */
#define PLA_B200_DEV_TABLE_FULL 64  /* a request needs more pages than its block-table row has columns */

/* Element strides of a paged cache tensor addressed [block, token in the block, head, channel]; channels contiguous. */
typedef struct pla_b200_page_strides {
  int64_t block, token, head;
} pla_b200_page_strides;

/* ======================================================================== *
 * Block tables and slot maps from request lengths, one launch.
 *   c = context_lens[n], m = query_start_loc[n + 1] - query_start_loc[n]
 *   held = ceil(c / block_size), need = min(ceil((c + m) / block_size), columns) - held (at least 0)
 *   block_table[n, held + j] = free_blocks[start + (sum of need before n) + j]
 * Token t of request n sits at position p = c + t - query_start_loc[n] and in slot
 * block_table[n, p / block_size] * block_size + p % block_size. Other entries of the table keep their values. Tokens at or past
 * query_start_loc[N], tokens without a page and tokens of a request with bad metadata (c < 0, m < 0, c + m past 32 bits, or an
 * offset query_start_loc[n] that is negative or below an earlier one: it takes no pages, seq_lens[n] = max(c, 0),
 * PLA_B200_DEV_BAD_INTERVAL) get slot -1; position 0 for the first and the last kind. A page past the end of the free
 * list becomes -1. `tokens` has to cover query_start_loc[N], which has to be the largest offset; new tokens past either are left
 * out of m, pages, table, seq_lens and free_next alike (PLA_B200_DEV_BAD_INTERVAL). Outputs must not overlap inputs
 * (block_table is both).
 * ======================================================================== */
typedef struct pla_b200_block_tables_args {
  int32_t* block_table;           /* [N, columns], pages of the context already in place */
  int64_t table_row_stride;       /* elements, >= columns */
  const int32_t* context_lens;    /* [N] tokens already in the cache */
  const int32_t* query_start_loc; /* [N + 1] offsets of the new tokens */
  const int32_t* free_blocks;     /* [free_count] */
  const int32_t* free_start;      /* [1] first entry of the list that is still free (below 0: 0), or NULL (0) */
  int64_t* slot_mapping;          /* [tokens] */
  int64_t* positions;             /* [tokens] */
  int32_t* seq_lens;              /* [N]: c + m */
  int32_t* free_next;             /* [1]: first entry that is free after this call, at most free_count */
  int32_t N, tokens, columns, free_count, block_size;
  int32_t* status;
} pla_b200_block_tables_args;

int pla_b200_block_tables(const pla_b200_block_tables_args* args, void* stream);

/* ======================================================================== *
 * Rotary positions over the first R channels of every head, after an optional per-head RMS norm, one launch:
 *   y = x * rsqrt(mean(x^2) + eps) * (w + unit_offset)           (when the weight is given)
 *   (y_a, y_b) <- factor * (y_a cos - y_b sin, y_b cos + y_a sin),  angle = position * inv_freq[i]
 * with (a, b) = (i, i + R/2), or (2i, 2i + 1) when interleaved. Angles are reduced to one turn in 64 bits; one rounding at the end.
 * k may be absent (Hk = 0). With k_cache (then k_out is NULL), k rows go to their slots and v rows
 * are copied to theirs; a slot < 0 stores nothing, a slot outside the pool sets PLA_B200_DEV_BAD_SLOT. Slots of one call
 * must differ. q_out / k_out may be q / k themselves; otherwise nothing that is written may overlap anything else. Rows and
 * strides are multiples of 16 bytes.
 * ======================================================================== */
typedef struct pla_b200_rotary_args {
  const void* q;       /* [T, Hq, D] */
  const void* k;       /* [T, Hk, D] */
  const void* v;       /* [T, Hk, D], with k_cache */
  int64_t q_tok_stride, q_head_stride, k_tok_stride, k_head_stride, v_tok_stride, v_head_stride;
  void* q_out;
  void* k_out;         /* NULL with k_cache */
  int64_t qo_tok_stride, qo_head_stride, ko_tok_stride, ko_head_stride;
  const void* q_weight; /* [D] or NULL (no norm of q) */
  const void* k_weight; /* [D] or NULL (no norm of k) */
  int32_t q_weight_dtype, k_weight_dtype;  /* any pla_b200_dtype */
  pla_b200_index positions;  /* [T] */
  const double* inv_freq;    /* [R / 2], radians per position */
  void* k_cache;
  void* v_cache;
  pla_b200_page_strides k_strides, v_strides;
  pla_b200_index slots;      /* [T], with k_cache */
  int64_t num_blocks;
  int32_t block_size;
  int32_t T, Hq, Hk, D, R;   /* D a multiple of 8, at most 256; R even, at most D */
  int32_t interleaved, unit_offset;
  int32_t act_dtype;         /* BF16 or F16 */
  float factor, eps;
  int32_t* status;
} pla_b200_rotary_args;

int pla_b200_rotary(const pla_b200_rotary_args* args, void* stream);

/* ======================================================================== *
 * Attention of one new token per request over a paged key/value cache:
 *   s_j = scale * q . k_j,  j < seq_lens[b];  lse = log(sum exp(s_j));  out = sum exp(s_j - lse) v_j
 * Query head h reads key/value head h / (Hq / Hk). A request of length 0 gets zeros and lse = -inf. Token j sits in page
 * block_table[b, j / block_size]. Tokens at or past seq_lens[b] never reach the result, but up to 15 rows behind it in the last
 * page may be read; table entries past the request's pages are not. A length < 0 (taken as 0) or past the table's columns or 2^30
 * (cut there) sets PLA_B200_DEV_BAD_INTERVAL; tokens whose page lies outside the pool are left out and set PLA_B200_DEV_BAD_SLOT.
 * NaN scores make the outputs and lse that they are part of NaN. `out` may be q itself when q is dense.
 * ======================================================================== */
typedef struct pla_b200_paged_decode_args {
  const void* q;        /* [B, Hq, D] */
  int64_t q_row_stride, q_head_stride;
  const void* k_cache;  /* [num_blocks, block_size, Hk, D] addressed with the strides */
  const void* v_cache;
  pla_b200_page_strides k_strides, v_strides;
  const int32_t* block_table; /* [B, columns] */
  int64_t table_row_stride;
  const int32_t* seq_lens;    /* [B] */
  void* out;            /* [B, Hq, D] dense, activation dtype */
  float* lse;           /* [B, Hq] or NULL */
  int64_t num_blocks;
  int32_t block_size, columns;
  int32_t B, Hq, Hk, D; /* D: 64, 96, 128, 192 or 256 */
  int32_t act_dtype;    /* BF16 or F16, of q, both caches and out */
  float scale;
  void* workspace;      /* device scratch of pla_b200_paged_decode_workspace_bytes() bytes, 16-byte aligned; used by this call alone,
                           any contents. May be NULL when that is 0 */
  int64_t workspace_bytes;
  int32_t* status;
} pla_b200_paged_decode_args;

/* Bytes for a call with these sizes (B, Hq, Hk, D, columns, block_size are read) on the current device, or a negative code. */
int64_t pla_b200_paged_decode_workspace_bytes(const pla_b200_paged_decode_args* args);
int pla_b200_paged_decode(const pla_b200_paged_decode_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* PLA_B200_ATTENTION_H_ */
