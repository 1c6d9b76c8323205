/*
 * spmm_attn.h -- C ABI of the attention operators (libspmm_attn.so): causal attention under a sliding window with a
 * few first keys that stay visible, its gradients, the form for one new token a sequence over keys and values held in
 * pages, and the write of new keys and values into those pages.
 *
 * They stand beside the pipeline's SDDMM -> softmax -> SpMM (spmm_pipeline.h): there the mask is any CSR pattern and
 * the weights pass through memory; here the mask is a band plus the first columns, given by two numbers, and neither
 * mask nor weights are stored.  For query i of a sequence with Lq queries and Lk keys, at position p = i + Lk - Lq:
 *
 *   visible(p, j) = j <= p  and  (window == 0  or  p - j < window  or  j < sinks)
 *   s[j] = scale * <q_i, k_j>,  lse = log sum_visible exp(s),  out = sum_visible exp(s - lse) v_j
 *
 * A query that sees no key (Lk < Lq) has out = 0, lse = -inf and gradients of 0.  What stands in places that a query
 * does not see, infinities and NaN included, does not reach its results.  A value that it sees and that is not finite is
 * added to out as it is, however small its weight.
 *
 * Query head h reads key/value head h / (heads / kv_heads).  Element types: SPMM_ATTN_F32, SPMM_ATTN_F16,
 * SPMM_ATTN_BF16; scores, softmax statistics and sums are 32-bit floats.  With the 16-bit types spmm_attn_window rounds
 * the weights to that type before they enter a product, and spmm_attn_window_grad the weights and their gradients where
 * they enter dv and dk; in dq and in spmm_attn_paged they enter as a rounded value plus its rounded remainder.  What is rounded
 * to float16 is scaled by powers of two first, so small weights, and gradients small or large, keep its bits.  Results
 * do not depend on anything but the arguments: no atomics, fixed orders of summation (in spmm_attn_paged the order is
 * a matter of all the lengths).
 *
 * Every pointer is a device address on `device`, and what a call writes does not overlap what it reads.  Calls are
 * ordered on `stream` (a hipStream_t, NULL = the null stream), hold no state between calls and can be captured in a
 * graph.  Calls that run at the same time need separate workspaces.  The current device is put back before a call
 * returns.  Status codes are the engine's (spmm_hip.h).
 */
#ifndef SPMM_ATTN_H
#define SPMM_ATTN_H

#include <stddef.h>
#include <stdint.h>

#include "spmm_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SPMM_ATTN_F32   SPMM_HIP_F32
#define SPMM_ATTN_F16   2
#define SPMM_ATTN_BF16  3

#define SPMM_ATTN_MAX_DIM    128   /* widest head */

typedef struct spmm_attn_desc {
    int32_t device, dtype;
    int32_t heads, kv_heads;      /* heads a multiple of kv_heads                                               */
    int32_t dim;                  /* head width, 1 .. SPMM_ATTN_MAX_DIM                                         */
    int32_t window, sinks;        /* window 0: no limit                                                         */
    float scale;                  /* times log2(e) finite                                                       */
    int64_t batch;                /* sequences                                                                  */
    int64_t q_len, k_len;         /* without offsets: rows of every sequence; with offsets: rows of the buffers */
    int32_t zero_rest;            /* with offsets: 1 = rows behind the last sequence are set to 0 in what the
                                     call writes (lse: -inf), 0 = they are left as they are                     */
    int32_t reserved;             /* 0 */
} spmm_attn_desc_t;

/* Rows of heads: element (sequence b, row t, head h, d) at ptr + b * seq + t * row + h * head + d (in elements).  With
 * offsets there is one sequence of rows and `seq` is not used.  Rows that are read may repeat (strides of 0); rows that
 * are written may not overlap. */
typedef struct spmm_attn_rows {
    void *ptr;
    int64_t seq, row, head;
} spmm_attn_rows_t;

/* Pages of a cache: row s of page g, key/value head h at k + g * k_page + s * k_row + h * k_head + d (v alike).
 * Position t of sequence b is row t % page_rows of page table[b * table_stride + t / page_rows].  lengths[b] positions
 * of sequence b are in the cache.  A table entry outside [0, pages) that a sequence needs, a negative length, or one
 * above table_cols * page_rows makes the attention of that sequence NaN and its append a no-op for those rows; entries
 * that no visible position needs are not read. */
typedef struct spmm_attn_pages {
    void *k, *v;
    int64_t pages, page_rows;
    int64_t k_page, k_row, k_head;
    int64_t v_page, v_row, v_head;
    const int32_t *table;         /* [batch][table_cols], rows table_stride apart */
    int64_t table_cols, table_stride;
    const int32_t *lengths;       /* [batch] */
} spmm_attn_pages_t;

/* Attention of whole sequences.  cu_q / cu_k: NULL (every sequence has q_len queries and k_len keys) or both int32
 * [batch + 1] offsets on the device: sequence b has rows cu[b] .. cu[b + 1] - 1, cu[0] = 0, not decreasing.
 * lse: float, [batch][q_len][heads] (with offsets [q_len][heads]), contiguous. */
int spmm_attn_window(const spmm_attn_desc_t *a, const spmm_attn_rows_t *q, const spmm_attn_rows_t *k,
                     const spmm_attn_rows_t *v, const int32_t *cu_q, const int32_t *cu_k, const spmm_attn_rows_t *out,
                     float *lse, void *stream);

/* Its gradients: dout with the forward pass's out and lse -> dq, dk, dv.  out and lse have to be what spmm_attn_window gave for
 * just these keys, not joined over further ones: that every query's row of score gradients sums to 0 is used to take the
 * rounding of out from dk.  `work`: spmm_attn_window_work bytes (packed: 1 = the call gives offsets), 16-byte aligned. */
int spmm_attn_window_work(const spmm_attn_desc_t *a, int32_t packed, size_t *bytes);
int spmm_attn_window_grad(const spmm_attn_desc_t *a, const spmm_attn_rows_t *dout, const spmm_attn_rows_t *q,
                          const spmm_attn_rows_t *k, const spmm_attn_rows_t *v, const spmm_attn_rows_t *out,
                          const float *lse, const int32_t *cu_q, const int32_t *cu_k, const spmm_attn_rows_t *dq,
                          const spmm_attn_rows_t *dk, const spmm_attn_rows_t *dv, void *work, size_t work_bytes,
                          void *stream);

/* One new token a sequence, which is the last of its lengths[b] positions: q and out have one row a sequence (`row` and
 * q_len, k_len are not used), lse is float [batch][heads].  max_length: no sequence is longer than this (one that is
 * counts as a bad length); it sizes the split of the work.  `work`: spmm_attn_paged_work bytes, 16-byte aligned. */
int spmm_attn_paged_work(const spmm_attn_desc_t *a, int64_t max_length, size_t *bytes);
int spmm_attn_paged(const spmm_attn_desc_t *a, const spmm_attn_rows_t *q, const spmm_attn_pages_t *pages,
                    int64_t max_length, const spmm_attn_rows_t *out, float *lse, void *work, size_t work_bytes,
                    void *stream);

/* Write new keys and values: the rows of sequence b go to its last positions, lengths[b] - n .. lengths[b] - 1.
 * cu NULL: one row a sequence (a padded sequence of length 0 writes nothing); otherwise offsets as above, with q_len
 * rows in the buffers.  Pages that are written must not be shared by two sequences.  heads, window, sinks and scale are
 * not used.  k and v may be NULL only if there are no rows. */
int spmm_attn_append(const spmm_attn_desc_t *a, const spmm_attn_rows_t *k, const spmm_attn_rows_t *v, const int32_t *cu,
                     const spmm_attn_pages_t *pages, void *stream);

const char *spmm_attn_last_error_detail(void);

#ifdef __cplusplus
}
#endif

#endif /* SPMM_ATTN_H */
