// attn_window.hpp -- arguments and index arithmetic of the window attention kernels (forward and gradients).
#pragma once
#include "attn_common.hpp"

namespace attn {

struct WindowArgs {
    Rows q, k, v, out, dout, dq, dk, dv;
    float *lse;              // forward: written; gradients: read
    float *stats;            // gradients: of every query row, laid out like lse, lse in powers of two and sum_d dout * out
    const int32_t *cu_q, *cu_k;
    int64_t batch, q_len, k_len;
    int heads, kv_heads, dim;
    Mask mask;
    float scale, scale2;     // scale2 = scale * log2(e): the exponentials are powers of two
    int tiles, zero_rest;
    float *part;             // gradients: parts of the first keys' gradients
    int chunk;               // queries of a part, 0: not split
    int block_keys;          // keys of a block of the kernel that owns keys
};

// Key head, query head inside its group, and tile of a block.  Consecutive blocks go round the eight dies, so
// consecutive blocks take different key heads: the blocks that share a key head's rows then mostly share a die's L2.
__device__ __forceinline__ void place(const WindowArgs &A, int inside, int *kv, int *g, int *tile) {
    const int per = A.kv_heads * inside, id = (int)blockIdx.x, hh = id % per;
    *kv = hh % A.kv_heads;
    *g = hh / A.kv_heads;
    *tile = id / per;
}

// Row 0 of a sequence and head.
template <typename T> __device__ __forceinline__ T *seq_base(const Rows &r, const Seq &s, int64_t first, bool packed, int head) {
    return (T *)r.ptr + (packed ? first * r.row : s.b * r.seq) + head * r.head;
}

// Rows [c, c + rows) for c = from, from + step, ... below end, of one head, set to zero: the blocks whose tile lies behind
// the last sequence share out the rows that no sequence has.
template <typename T> __device__ void zero_rows(const Rows &r, int64_t from, int64_t step, int rows, int64_t end, int head,
                                                int dim) {
    for (int64_t c = from; c < end; c += step)
        for (int i = threadIdx.x; i < rows * dim; i += blockDim.x) {
            const int64_t row = c + i / dim;
            if (row < end) ((T *)r.ptr)[row * r.row + head * r.head + i % dim] = (T)0.f;
        }
}

// row of register r (+ 4 h) in a 32x32 product
__device__ __forceinline__ constexpr int row_of(int r) { return 8 * (r >> 2) + (r & 3); }

template <typename T> __device__ __forceinline__ frag<T> next_operand(const f32x16 &c, int ks);

// acc += tile^T w over a tile of ROWS rows some value of which is not finite; w: weights of the tile's rows for the lane's
// column, 0 where seen(row) does not hold.  A masked place enters the matrix instructions as 0 * x, which is NaN for such
// an x: it is taken out of the operand and put back where it is seen.  Rare, so a function of its own that takes no
// registers from the loops that call it.
template <typename T, int DP, int ROWS> struct Careful {
    f32x16 acc[DP / 32], w[ROWS / 32];
};
// BOTH: what rounding w to the type leaves enters as well, after it.
template <typename T, int DP, int ROWS, bool BOTH = false>
__device__ __attribute__((noinline)) void careful_product(Careful<T, DP, ROWS> *c, const T *tile, int lane, Mask mask, int p, int j0,
                                                          bool by_key, int last) {
#pragma unroll 1
    for (int n = 0; n < ROWS / 32; ++n)
#pragma unroll 1
        for (int k2 = 0; k2 < 2; ++k2) {
            frag<T> pf, low;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                pf[j] = narrow<T>(c->w[n][8 * k2 + j]);
                low[j] = narrow<T>(c->w[n][8 * k2 + j] - (float)pf[j]);
            }
#pragma unroll 1
            for (int d = 0; d < DP / 32; ++d) {
                frag<T> f = Tile<T, DP>::col_frag(tile, n * 32 + k2 * 16, d * 32, lane);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!finite_f((float)f[j])) f[j] = (T)0.f;
                c->acc[d] = mma32(f, pf, c->acc[d]);
                if (BOTH) c->acc[d] = mma32(f, low, c->acc[d]);
            }
        }
    if (last < j0) return;
#pragma unroll 1
    for (int rr = 0; rr < ROWS; ++rr) {
        // rows are keys and the column a query at p, or rows are queries at j0 + rr and the column key p
        const bool seen = j0 + rr <= last && (by_key ? mask.sees(p, j0 + rr) : mask.sees(j0 + rr, p));
#pragma unroll 1
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float x = (float)tile[Tile<T, DP>::at(rr, d * 32 + 8 * (r >> 2) + (r & 3) + 4 * (lane >> 5))];
                if (seen && !finite_f(x)) c->acc[d][r] += x;
            }
    }
}

// acc += the values that are not finite of the keys from `from` to `to` that the lane's query, at position p, sees; a lane has the
// elements of a result's column that the products give it.  Without their weights: a weight is positive, but may be rounded
// to 0, in which case a product would make NaN of an infinity.  64 lanes look a row over, eight rows on their way at a time.
template <typename T, int DP> struct Sums {
    f32x16 acc[DP / 32];
};
template <typename T, int DP>
__device__ __attribute__((noinline)) void add_not_finite_rows(Sums<T, DP> *c, const T *v, int64_t row, int dim, int lane, Mask mask,
                                                              int p, int from, int to) {
#pragma unroll 1
    for (int j0 = from; j0 <= to; j0 += 8) {
        float x[8][2];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int s = 0; s < 2; ++s)
                x[i][s] = j0 + i <= to && lane + 64 * s < dim ? (float)v[(int64_t)(j0 + i) * row + lane + 64 * s] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int s = 0; s < 2; ++s)
                for (unsigned long long m = __ballot(!finite_f(x[i][s])); m; m &= m - 1) {
                    const int el = __ffsll(m) - 1, e = el + 64 * s;
                    const float y = __shfl(x[i][s], el);
                    if ((lane >> 5) == (e >> 2 & 1) && mask.sees(p, j0 + i)) c->acc[e >> 5][(e >> 3 & 3) * 4 + (e & 3)] += y;
                }
    }
}

// registers 8 ks .. 8 ks + 7 of a product as the next product's operand (rows 16 ks + ... in col_frag's order)
template <typename T> __device__ __forceinline__ frag<T> next_operand(const f32x16 &c, int ks) {
    frag<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = narrow<T>(c[8 * ks + j]);
    return f;
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}
int window_args(const spmm_attn_desc_t *a, const char *where, const int32_t *cu_q, const int32_t *cu_k, WindowArgs *out);
int tile_count(const spmm_attn_desc_t *a, const char *where, bool packed, int64_t len, int rows, int *tiles);

}  // namespace attn
