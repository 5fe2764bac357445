/*
 * ztcp_kvcache.h -- operators on the hot side of the paged KV pool (libztcp_b200.so): what fills the pages that
 * egress encrypts, reads the pages that ingress restores, and chooses the pages that leave the pool.
 *
 * The reference (research/baseline_codec) has no operator of this kind: it encodes and decodes pages that a
 * serving engine owns.  The pool, page and block-table conventions are those of ztcp_b200.h: a page is
 * num_tokens x num_heads x head_dim elements per buffer, dense, fp16 or bf16; v_pool = NULL is a single-buffer
 * (MLA) pool whose values are columns [rope_dim, head_dim) of K.
 *
 *   ztcp_append_tokens      norms of queries and keys per head + position rotation + write into pool slots
 *   ztcp_attend_pages       attention of the sequences' newest tokens over their pages, with the log-sum-exp
 *   ztcp_page_mass          attention weight of those tokens, accumulated per page
 *   ztcp_select_cold_pages  the pages with the least weight, as a block table for ztcp_encode_pages, and the
 *                           compacted tables of the pages that stay
 *
 * Every call only enqueues work on `stream` and returns ZTCP_OK, or a negative code with a message from
 * ztcp_last_error().  No call allocates memory or synchronizes; every call can be captured into a CUDA graph.
 * Every pointer is device memory of the current device.  Lengths, tables and slots are read on the device at
 * every call and checked there before they address memory: a bad one is never followed, and is reported in
 * `status`.
 * A batch holds at least one sequence, query row or token; an empty one is refused.
 */
#ifndef ZTCP_KVCACHE_H
#define ZTCP_KVCACHE_H

#include <stdint.h>

#include "ztcp_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Status of a sequence (or of an appended token), int32: */
#define ZTCP_SEQ_OK 0
#define ZTCP_SEQ_BAD_LENGTH 5 /* kv_lens outside [0, max_pages * num_tokens] or beyond 2^31 - 4096, or q_starts not ascending within
                                 [0, total_rows]: clamped to that range */
#define ZTCP_SEQ_BAD_BLOCK 6  /* a block-table entry outside the pool: its page counts as masked; append: a slot
                                 or position out of range: the token is not written */
#define ZTCP_SEQ_TIMEOUT 7    /* a wait inside the attention kernel did not end: the outputs are not valid */

/* A paged KV cache as n_seqs sequences see it.  Sequence b holds kv_lens[b] tokens (its newest ones included);
 * token j lies in page block_tables[b * table_stride + j / num_tokens], row j % num_tokens.  Entries past the
 * last page are not read.  K and V rows below kv_lens[b] must be finite. */
typedef struct ztcp_kv_cache {
  const void* k_pool;          /* [pool_pages, num_tokens, num_heads, head_dim], 16-byte aligned */
  const void* v_pool;          /* same, or NULL: values are columns [rope_dim, head_dim) of K */
  int32_t dtype;               /* ZTCP_DTYPE_* of the pools, the queries and the output */
  int32_t reserved;
  ztcp_geometry geom;          /* num_heads = KV heads; is_mla_single_buffer is not read */
  int64_t pool_pages;
  const int32_t* block_tables; /* [n_seqs, table_stride] */
  int64_t table_stride;
  int64_t max_pages;           /* entries of a row that may be read */
  const int32_t* kv_lens;      /* [n_seqs] */
  int64_t n_seqs;              /* 1 to 2^21 */
} ztcp_kv_cache;

/* The newest tokens' queries, packed: sequence b owns rows [q_starts[b], q_starts[b + 1]).  Its row i is token
 * kv_len - q_len + i; with `causal` it sees tokens up to itself, otherwise all of the sequence.  A row that sees
 * nothing gets a zero output and a log-sum-exp of -inf.  Where starts do not ascend, rows that two sequences claim get the
 * result of either. */
typedef struct ztcp_queries {
  const void* q;            /* row r, head h at q + r * token_stride + h * head_stride elements; 16-byte aligned */
  int64_t token_stride;     /* elements, multiples of 8 */
  int64_t head_stride;
  const int32_t* q_starts;  /* [n_seqs + 1], or NULL: one row per sequence (total_rows = n_seqs) */
  int64_t total_rows;
  int64_t num_heads;        /* a multiple of the KV heads; query head h reads KV head h / (num_heads / KV heads) */
  int64_t max_q_len;        /* longest q_len to expect (below 2^31): chooses the kernel; any q_len is computed */
  float scale;              /* of the scores: positive, finite times log2(e) */
  int32_t causal;
} ztcp_queries;

/* Workspace bytes of ztcp_attend_pages on the current device; -1 when the arguments are invalid. */
int64_t ztcp_attend_workspace_bytes(const ztcp_kv_cache* cache, const ztcp_queries* queries);

/* out [total_rows, num_heads, value columns] (dtype), lse [total_rows, num_heads] fp32 or NULL (natural
 * logarithm of the sum of exp(scale * score)), status [n_seqs] int32.  Rows behind the last sequence are left as
 * they were.  head_dim up to 256, or up to 576 with at most 512 value columns when v_pool is NULL.
 * `workspace`: device memory of at least ztcp_attend_workspace_bytes, 16-byte aligned, needing no
 * initialisation; calls that may run at the same time need one each. */
int32_t ztcp_attend_pages(const ztcp_kv_cache* cache, const ztcp_queries* queries, void* out, float* lse,
                          int32_t* status, void* workspace, int64_t workspace_bytes, void* stream);

/* Workspace bytes of ztcp_page_mass on the current device; -1 when the arguments are invalid. */
int64_t ztcp_page_mass_workspace_bytes(const ztcp_kv_cache* cache, const ztcp_queries* queries);

/* out_mass[b, p] = decay * mass[b, p] + sum over the sequence's rows, their heads and the tokens j of page p that
 * the row sees, of exp(scale * score - lse[row, head]); 0 past the sequence's last page.  mass and out_mass are
 * [n_seqs, max_pages] fp32, dense, and may be the same memory; mass may be NULL (no earlier weight).  lse as
 * ztcp_attend_pages writes it; a row whose lse is -inf adds nothing.  `workspace`: as for ztcp_attend_pages. */
int32_t ztcp_page_mass(const ztcp_kv_cache* cache, const ztcp_queries* queries, const float* lse, const float* mass,
                       float decay, float* out_mass, int32_t* status, void* workspace, int64_t workspace_bytes,
                       void* stream);

/* Norm, rotation and append of new tokens.  Row r of q (num_q_heads vectors) goes to q_out (dense), of k and v
 * (geom.num_heads vectors each) to pool slot slots[r] (page slots[r] / num_tokens, row slots[r] % num_tokens); a
 * slot of -1 writes no K/V.  Slots must be distinct.  Per q and k vector x: with a weight w, columns
 * [norm_from, head_dim) become x * w / sqrt(mean(x^2 over those columns) + eps); then columns [0, rope_dim) are
 * rotated by row positions[r] of the table (cosines in its first rope_dim / 2 columns, sines in the others),
 * column i paired with i + rope_dim / 2, or 2i with 2i + 1 when interleaved.  v is copied.  The arithmetic is
 * fp32, rounded once.  A token whose position lies outside [0, max_pos) or whose slot lies outside the pool is
 * reported in status[r]; the former writes nothing, the latter its query only.  q may equal q_out. */
typedef struct ztcp_append {
  const void *q, *k, *v;      /* rows, as ztcp_queries; v NULL exactly when v_pool is; q NULL: no queries */
  int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride;
  void* q_out;                /* [n_tokens, num_q_heads, head_dim] */
  void *k_pool, *v_pool;
  const int64_t* slots;       /* [n_tokens] */
  const int32_t* positions;   /* [n_tokens] */
  const float* rope_table;    /* [max_pos, rope_dim], 16-byte aligned; NULL when rope_dim is 0 */
  const float *q_weight, *k_weight; /* [head_dim - norm_from] fp32, 16-byte aligned, or NULL: no norm */
  int64_t n_tokens, num_q_heads, pool_pages, max_pos;
  ztcp_geometry geom;
  int32_t dtype, norm_from, interleaved;
  float eps;
} ztcp_append;

int32_t ztcp_append_tokens(const ztcp_append* a, int32_t* status, void* stream);

/* Choice of the pages to evict.  Sequence b has n = ceil(kv_lens[b] / page_tokens) pages; of pages
 * [sink, n - recent) the min(n - keep, n - recent - sink) (at least 0) with the least mass are cold, ties going to
 * the lower page; a NaN counts as more than any number.  recent is at least 1: the last page, which may be
 * partly filled, always stays.
 *   cold_starts [n_seqs + 1], cold_blocks / cold_index [n_seqs * max_pages]: sequence b's cold pages, ascending,
 *     at [cold_starts[b], cold_starts[b + 1]): their pool blocks (a kv_block table for ztcp_encode_pages) and
 *     b * max_pages + page; -1 behind the last
 *   kept_tables / kept_mass [n_seqs, max_pages]: the other pages in order, then -1 / 0
 *   kept_lens [n_seqs]: kv_lens minus the cold pages' tokens
 * The outputs overlap neither each other nor the inputs.  A kv_len outside [0, max_pages * page_tokens] is clamped to
 * it and reported.  n_seqs * max_pages is below 2^31, and max_pages at most 2^31 - 4096. */
typedef struct ztcp_cold_selection {
  const float* mass;           /* [n_seqs, max_pages] */
  const int32_t* block_tables; /* [n_seqs, max_pages] */
  const int32_t* kv_lens;
  int64_t n_seqs, max_pages, page_tokens, keep, sink, recent;
  int32_t *cold_blocks, *cold_index, *cold_starts, *kept_tables;
  float* kept_mass;
  int32_t *kept_lens, *status;
} ztcp_cold_selection;

int32_t ztcp_select_cold_pages(const ztcp_cold_selection* s, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ZTCP_KVCACHE_H */
