/*
 * spmm_q4.h -- C ABI of products with 4-bit weights (libspmm_q4.so): y = x W^T for a few rows of x, the K = 1 product's
 * counterpart (spmm_pbv.h) for weights that are compressed to 4 bits instead of pruned.
 *
 *   y[t][n] = sum_k x[t][k] w[n][k],   w[n][k] = scale[n][k / group] * (q[n][k] - zero[n][k / group])
 *
 * q: 4-bit numbers 0 .. 15; zero: 8 without zero points.  x, y and the scales have one element type: SPMM_Q4_F32,
 * SPMM_Q4_F16 or SPMM_Q4_BF16.  Weights enter the products exactly (q + 16 in 16 bits), x as it is (32-bit x as three
 * 16-bit parts that sum to it); sums are 32-bit floats in a fixed order, and y is rounded once.  The products are formed with
 * 16 + q and 16 + zero over up to 128 columns at a time, and those are subtracted: an infinite x gives NaN, and so may finite
 * ones of which such a sum, up to 31 times that of x, passes 32-bit floats (from 1.1e37 in one column, 8.5e34 in 128, on).
 *
 * The weights are laid out once (spmm_q4_layout) in the order in which the product's waves read them; the product reads
 * only the layout.  Every pointer is a device address on `device`, y does not overlap what is read, calls are ordered on `stream`, hold no state and
 * can be captured in a graph.  The current device is put back before a call returns.  Status codes are the engine's.
 */
#ifndef SPMM_Q4_H
#define SPMM_Q4_H

#include <stddef.h>
#include <stdint.h>

#include "spmm_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SPMM_Q4_F32   SPMM_HIP_F32
#define SPMM_Q4_F16   2
#define SPMM_Q4_BF16  3

typedef struct spmm_q4_desc {
    int32_t device, dtype;
    int64_t rows, cols;      /* of W                                                                         */
    int32_t group;           /* columns that share a scale: 32, 64 or a multiple of 128; the last may be short */
    int32_t zeros;           /* 1: zero points are given                                                     */
} spmm_q4_desc_t;

/* Bytes of the layout. */
int spmm_q4_layout_bytes(const spmm_q4_desc_t *w, size_t *bytes);

/* packed: uint8 [rows][(cols + 1) / 2], column 2 i in the low half of byte i, rows packed_stride bytes apart; scales:
 * [rows][groups], rows scale_stride elements apart, groups = cols / group rounded up; zeros: uint8 [rows][groups], rows
 * zero_stride apart (NULL without zero points).  dst: the layout, 256-byte aligned. */
int spmm_q4_layout(const spmm_q4_desc_t *w, const void *packed, int64_t packed_stride, const void *scales,
                   int64_t scale_stride, const void *zeros, int64_t zero_stride, void *dst, size_t dst_bytes, void *stream);

/* x: [tokens][cols], rows x_stride elements apart (0: one row for all); y: [tokens][rows], rows y_stride apart. */
int spmm_q4_matvec(const spmm_q4_desc_t *w, const void *layout, const void *x, int64_t x_stride, int64_t tokens, void *y,
                   int64_t y_stride, void *stream);

const char *spmm_q4_last_error_detail(void);

#ifdef __cplusplus
}
#endif

#endif /* SPMM_Q4_H */
