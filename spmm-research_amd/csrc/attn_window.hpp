// attn_window.hpp -- arguments and index arithmetic of the window attention kernels (forward and gradients).
#pragma once
#include "attn_common.hpp"

namespace attn {

struct WindowArgs {
    Rows q, k, v, out, dout, dq, dk, dv;
    float *lse;              // forward: written; gradients: read
    float *delta;            // gradients: sum_d dout * out of every query row, laid out like lse
    const int32_t *cu_q, *cu_k;
    int64_t batch, q_len, k_len;
    int heads, kv_heads, dim;
    Mask mask;
    float scale, scale2;     // scale2 = scale * log2(e): the exponentials are powers of two
    int tiles, zero_rest;
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

// acc[d][r] += the tile's values that are not finite and stand in a row that the lane's column sees.  A masked place
// enters the matrix instructions as 0 * x, which is NaN for such an x: it is taken out of the operand (only_finite)
// and put back here where it is seen.
template <typename T, int DP, typename F>
__device__ __forceinline__ void add_not_finite(f32x16 (&acc)[DP / 32], const T *tile, int rows, int lane, F sees) {
#pragma unroll 1
    for (int rr = 0; rr < rows; ++rr) {
        const bool seen = sees(rr);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float x = (float)tile[Tile<T, DP>::at(rr, dt * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3))];
                if (seen && !finite_f(x)) acc[dt][r] += x;
            }
    }
}
template <typename T> __device__ __forceinline__ frag<T> only_finite(frag<T> f) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (!finite_f((float)f[j])) f[j] = (T)0.f;
    return f;
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
// row of register r (+ 4 h) in a 32x32 product
__device__ __forceinline__ constexpr int row_of(int r) { return 8 * (r >> 2) + (r & 3); }

int window_args(const spmm_attn_desc_t *a, const char *where, const int32_t *cu_q, const int32_t *cu_k, WindowArgs *out);
int tile_count(const spmm_attn_desc_t *a, const char *where, bool packed, int64_t len, int rows, int *tiles);

}  // namespace attn
