// attn_window.hip -- causal attention under a sliding window with first keys that stay visible (include/spmm_attn.h).
//
// One pass over the keys with a running maximum and sum.  A workgroup has four waves of 32 queries each of one head; the
// keys and values that its 128 queries see come by tiles through LDS.  Scores are formed transposed, S^T = K Q^T, so a
// lane owns one query (column l % 32) and half of the tile's keys: the softmax statistics of a query need one exchange
// between two lanes, and S^T leaves the matrix unit in the layout in which exp(S^T) is the second operand of
// O^T = V^T P^T -- the weights never pass through LDS.  V^T comes from the row-major tile by the transposing LDS read.
//
// A value that is not finite, if it is seen, is added to the result as it is: the block starts over, leaves such values out of
// the products, and adds them at the end.  That none stands where it would show costs a look at the sums and a barrier a
// block: 8192 tokens, window 1024, 32 heads over 8 of 128 in bf16 190 us from 188.  With an infinity that all see, 16384 tokens
// under a window of 2048 take 15.5 ms, and 4.0 with one in the middle.
//
// The weights of 16-bit types are rounded to the type for the second product, at most 2^-8 (bf16) or 2^-11 (fp16) of each,
// as the values are; their sum is taken before that, in 32 bits.  The result's error against float64 is then 1.4 (bf16) and 1.2
// (fp16) times that of its own rounding.  As a rounded value plus its remainder they would enter half as many products more:
// 794 us for the 608 of the 16384 tokens below, 460 for 366 of 8192 and 8000 under a window of 1024.
//
// Bound: matrix instructions and the exponentials beside them, which do not overlap within a wave; two blocks a compute
// unit fill the gaps of each other.  One sequence of 16384 tokens, 32 heads over 8 of 128 in bf16, window 2048, 16 first
// keys: 608 to 629 us in six runs, 825 to 850 TFLOP/s of products (a plain product of 8192^3 reaches 1127); the matrix units
// are busy for 40 % of the cycles, the vector units for 46, LDS for 21.  128 queries a block: with 256 (eight waves) 699 to
// 728 us.  Loading the next tile's fragments ahead, unrolling by two tiles and raised wave priority gained nothing.  A ragged
// batch of eight of 0 to 2051 tokens, 16 heads over 4 of 80, window 256: 38 us, with 64 queries a block 41 to 48; its 560 blocks
// of up to eight tiles each meet 512 places, so 48 run after the others.
#include "attn_window.hpp"

namespace attn {

// How a block is made up: MG groups of 32 queries times PG waves that share a group's keys, 32 SUB of every tile each, and
// join at the end; two tiles of 32 PG SUB keys on their way or in use.
template <typename T, int DP, int MG, int PG, int SUB> struct WindowShape {
    static constexpr int ROWS = 32 * MG, BN = 32 * PG * SUB, THREADS = 64 * MG * PG;
};
constexpr int SLACK = 8;

template <typename T, int DP, int MG, int PG, int SUB, bool DIRECT>
__global__ __launch_bounds__(64 * MG * PG, sizeof(T) == 2 && PG == 1 ? 2 : 1) void window_kernel(WindowArgs A) {
    using L = Tile<T, DP>;
    using S = WindowShape<T, DP, MG, PG, SUB>;
    constexpr int BM = S::ROWS, BN = S::BN, THREADS = S::THREADS, ND = DP / 32, NS = DP / 16, NK = SUB;
    constexpr float LIFT = UP<T>(SLACK);             // weights and their sum are 2^LIFT times as large
    __shared__ __align__(16) T sk[2][BN * L::PITCH], sv[2][BN * L::PITCH];
    __shared__ float sm[PG > 1 ? PG * MG * 32 : 1];  // the parts' maxima
    __shared__ int odd[2];                           // a value of the partly seen tile in this pair is not finite

    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5;
    const int mg = wave % MG, part = wave / MG;      // the wave's queries, and which keys of a tile
    int kv, g, t;
    place(A, A.heads / A.kv_heads, &kv, &g, &t);
    t = A.tiles - 1 - t;                             // late queries see more keys: they start first
    const int head = kv * (A.heads / A.kv_heads) + g;
    const bool packed = A.cu_q != nullptr;
    const Seq s = find_tile(t, BM, false, A.cu_q, A.cu_k, A.batch, A.q_len, A.k_len);
    if (s.tile < 0) {
        if (A.zero_rest && packed) {
            const int64_t from = s.rest + (int64_t)(t - s.nq) * BM, step = (int64_t)(A.tiles - s.nq) * BM;
            zero_rows<T>(A.out, from, step, BM, A.q_len, head, A.dim);
            for (int64_t c = from; c < A.q_len; c += step)
                for (int64_t r = c + tid; r < c + BM && r < A.q_len; r += blockDim.x) A.lse[r * A.heads + head] = -INFINITY;
        }
        return;
    }
    if (tid == 0) odd[0] = odd[1] = 0;

    const int shift = s.nk - s.nq, m0 = s.tile * BM, m1 = min(m0 + BM, s.nq) - 1;
    const int pmin = m0 + shift, pmax = m1 + shift;                       // positions of the block's queries
    const int lo = A.mask.window ? max(0, pmin - A.mask.window + 1) : 0;  // first key that the window holds
    const int lt = lo / BN, ht = pmax >= 0 ? pmax / BN : -1;
    const int ns = pmax >= 0 ? min((min(A.mask.sinks, pmax + 1) + BN - 1) / BN, lt) : 0;      // tiles of first keys before
    const int tiles = ns + max(0, ht - lt + 1);
    auto tile_at = [&](int i) { return (i < ns ? i : lt + i - ns) * BN; };

    const T *kb = seq_base<T>(A.k, s, s.k0, packed, kv), *vb = seq_base<T>(A.v, s, s.k0, packed, kv);
    const int i = m0 + mg * 32 + (lane & 31), p = i + shift;              // this lane's query
    const bool mine = i < s.nq;
    const int w0 = m0 + mg * 32 + shift, w1 = min(w0 + 31, pmax);         // the wave's positions
    frag<T> qf[NS];
    {
        const T *qr = mine ? seq_base<T>(A.q, s, s.q0, packed, head) + i * A.q.row : nullptr;
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            qf[st] = load_frag<T>(qr, st * 16 + h * 8, A.dim, A.q.wide);
            // the largest score is then the largest product, and a masked product of -inf stays one
            if (A.scale2 < 0.f) qf[st] = -qf[st];
            if (A.scale2 == 0.f) qf[st] = frag<T>{};
        }
        settled<T>(qf);
    }
    const float scale2 = A.scale2 == 0.f ? 1.f : fabsf(A.scale2);

    using Move = Mover<T, DP, BN, THREADS>;
    Move mk, mv;
    if (DIRECT) {
        mk.start(tid, A.dim, A.k.row);
        mv.start(tid, A.dim, A.v.row);
    }
    auto send = [&](int j0, T *tk, T *tv) {
        mk.send(wave, tk, kb + (int64_t)j0 * A.k.row, A.k.row, pmax + 1 - j0, A.dim);
        mv.send(wave, tv, vb + (int64_t)j0 * A.v.row, A.v.row, pmax + 1 - j0, A.dim);
    };
    // the tile is in LDS but for a barrier
    auto settle = [&](int j0, int buf, T *tk, T *tv) {
        if constexpr (DIRECT) {
            arrived();
        } else {
            auto copy = [&](T *tile, const T *base, int64_t row) {
                Move::copy(tid, A.dim, tile, [&](int r) { return j0 + r <= pmax ? base + (int64_t)(j0 + r) * row : nullptr; });
            };
            copy(tk, kb, A.k.row);
            copy(tv, vb, A.v.row);
        }
        if (!A.mask.all(pmin, pmax, j0, j0 + BN - 1) && Move::any_not_finite(tid, tv)) odd[buf] = 1;
    };

    f32x16 o[ND];
    float m, sum;                                    // of the scores times scale2
    auto step = [&](auto careful, int j0, const T *tk, const T *tv) {
        // A wave whose queries see none of the block's tile goes through it all the same: a way round it would have the
        // accumulators copied at the end of every turn.
        const bool full = A.mask.all(w0, w1, j0, j0 + 32 * SUB - 1);
        f32x16 sc[NK];
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            sc[n] = zero16();
#pragma unroll
            for (int st = 0; st < NS; ++st)
                sc[n] = mma32(L::row_frag(tk, n * 32 + (lane & 31), st * 16 + h * 8), qf[st], sc[n]);
        }
        if (!full) {
            asm volatile("");                        // a branch, not 32 selects in every tile
#pragma unroll
            for (int n = 0; n < NK; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!A.mask.sees(p, j0 + n * 32 + row_of(r) + 4 * h)) sc[n][r] = -INFINITY;
        }
        float mx = sc[0][0];
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[n][r]);
        mx = fmaxf(mx, __shfl_xor(mx, 32)) * scale2;
        // The exponentials' base follows the maximum only when that has grown by more than SLACK: weights up to
        // 2^SLACK lose nothing in any of the types, and the accumulators are rarely rescaled.
        // Each query by itself: its result then does not depend on which others share its wave.
        const bool grown = mx > m + SLACK;
        if (__any(grown)) {
            const float top = grown ? mx : m;
            const float alpha = grown ? __builtin_amdgcn_exp2f(m - top) : 1.f;
            sum *= alpha;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= alpha;
            m = top;
        }
        const float base = (m == -INFINITY ? 0.f : m) - LIFT;
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                sc[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][r], scale2, -base));
                sum += sc[n][r];
            }
        if constexpr (!careful) {
#pragma unroll
            for (int n = 0; n < NK; ++n)
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2) {
                    const frag<T> pf = next_operand<T>(sc[n], k2);
#pragma unroll
                    for (int d = 0; d < ND; ++d)
                        o[d] = mma32(L::col_frag(tv, n * 32 + k2 * 16, d * 32, lane), pf, o[d]);
                }
        } else {
            Careful<T, DP, 32 * SUB> c;
            for (int d = 0; d < ND; ++d) c.acc[d] = o[d];
            for (int n = 0; n < NK; ++n) c.w[n] = sc[n];
            careful_product<T, DP, 32 * SUB>(&c, tv, lane, A.mask, p, j0, true, -1);
            for (int d = 0; d < ND; ++d) o[d] = c.acc[d];
        }
    };

    // All tiles in turn; false if a value in a partly seen one is not finite and `careful` does not allow for that.  With
    // `careful` such values are left out, and added after everything else.
    auto run = [&](auto careful) {
        m = -INFINITY;
        sum = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = zero16();
        if (tiles) {
            if (DIRECT) send(tile_at(0), sk[0], sv[0]);
            settle(tile_at(0), 0, sk[0], sv[0]);
        }
        __syncthreads();
        for (int it = 0; it < tiles; ++it) {         // a tile's loads are under way while the one before it is used
            const int buf = it & 1, j0 = tile_at(it);
            // The whole block leaves at the same tile: what a wave ahead finds in the next one goes to the other flag.
            if (!careful && !A.mask.all(pmin, pmax, j0, j0 + BN - 1) && uniform(odd[buf])) return false;
            const bool more = it + 1 < tiles;
            if (DIRECT && more) send(tile_at(it + 1), sk[buf ^ 1], sv[buf ^ 1]);
            step(careful, j0 + 32 * SUB * part, sk[buf] + 32 * SUB * part * L::PITCH, sv[buf] + 32 * SUB * part * L::PITCH);
            if (more) settle(tile_at(it + 1), buf ^ 1, sk[buf ^ 1], sv[buf ^ 1]);
            __syncthreads();
        }
        return true;
    };
    __syncthreads();                                 // `odd` is set
    bool careful = !run(std::false_type{});          // the whole block leaves at the same tile
    if (!careful) {
        // Of a wholly seen tile such a value got its weight, and NaN where that was rounded to 0, then or in a rescaling.
        float zero = 0.f;                            // infinities and NaN times 0 are NaN
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) zero = __builtin_fmaf(o[d][r], 0.f, zero);
        // Not where the query's weights are NaN: its result is then.  odd[0] is 0: no tile has left with it set.
        if (zero != 0.f && finite_f(sum + __shfl_xor(sum, 32)) && mine) odd[0] = 1;
        __syncthreads();
        careful = uniform(odd[0]);
    }
    if (careful) {
        __syncthreads();
        run(std::true_type{});
    }
    sum += __shfl_xor(sum, 32);
    if constexpr (PG > 1) {                          // the parts, in order, through the tiles' place in LDS
        float *mail = reinterpret_cast<float *>(sk) + mg * ND * 16 * 64 + lane;
        sm[(part * MG + mg) * 32 + (lane & 31)] = m;
        __syncthreads();
        float top = m;
#pragma unroll
        for (int q = 0; q < PG; ++q) top = fmaxf(top, sm[(q * MG + mg) * 32 + (lane & 31)]);
        const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
        m = top;
        sum *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] *= f;
#pragma unroll 1
        for (int from = 1; from < PG; ++from) {
            if (from > 1) __syncthreads();
            if (part == from) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) mail[(d * 16 + r) * 64] = o[d][r];
            }
            __syncthreads();
            if (part == 0) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] += mail[(d * 16 + r) * 64];
            }
        }
        __syncthreads();
        sm[(part * MG + mg) * 32 + (lane & 31)] = sum;
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int q = 0; q < PG; ++q) sum += sm[(q * MG + mg) * 32 + (lane & 31)];
    }
    if (part != 0) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] *= inv;
    if (careful) {
        Sums<T, DP> c;
        const int from = A.mask.window ? max(0, w0 - A.mask.window + 1) : 0;
        for (int d = 0; d < ND; ++d) c.acc[d] = o[d];
        add_not_finite_rows<T, DP>(&c, vb, A.v.row, A.dim, lane, A.mask, p, 0, min(min(A.mask.sinks, from) - 1, w1));
        add_not_finite_rows<T, DP>(&c, vb, A.v.row, A.dim, lane, A.mask, p, from, w1);
        for (int d = 0; d < ND; ++d) o[d] = c.acc[d];
    }
    if (!mine) return;
    T *dst = seq_base<T>(A.out, s, s.q0, packed, head) + i * A.out.row;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            store4<T>(dst, d * 32 + row_of(r) + 4 * h, A.dim, A.out.wide,
                      f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]});
    if (h == 0) {
        const int64_t row = packed ? s.q0 + i : s.b * A.q_len + i;
        A.lse[row * A.heads + head] = sum == 0.f ? -INFINITY : (m - LIFT) * LN2 + __logf(sum);
    }
}

int window_args(const spmm_attn_desc_t *a, const char *where, const int32_t *cu_q, const int32_t *cu_k, WindowArgs *out) {
    if (!cu_q != !cu_k) return fail(SPMM_HIP_ERR_ARG, "%s: offsets for only one of queries and keys", where);
    if (((uintptr_t)cu_q | (uintptr_t)cu_k) % 4) return fail(SPMM_HIP_ERR_ARG, "%s: offsets are not aligned", where);
    *out = WindowArgs{};
    out->cu_q = cu_q;
    out->cu_k = cu_k;
    out->batch = a->batch;
    out->q_len = a->q_len;
    out->k_len = a->k_len;
    out->heads = a->heads;
    out->kv_heads = a->kv_heads;
    out->dim = a->dim;
    // a window over every key is no window; first keys beyond the last are none
    out->mask.window = a->window >= a->k_len ? 0 : a->window;
    out->mask.sinks = out->mask.window ? (int)(a->sinks < a->k_len ? a->sinks : a->k_len) : 0;
    out->scale = a->scale;
    out->scale2 = a->scale * LOG2E;
    out->zero_rest = a->zero_rest;
    return SPMM_HIP_OK;
}

// Tiles over all sequences: with offsets a bound that holds for any lengths of that sum, and one more, which lies behind
// the last sequence, where rows there are to be set.
int tile_count(const spmm_attn_desc_t *a, const char *where, bool packed, int64_t len, int rows, int *tiles) {
    const int64_t n = packed ? len / rows + a->batch + (a->zero_rest ? 1 : 0) : a->batch * ((len + rows - 1) / rows);
    if (n > INT32_MAX / a->heads) return fail(SPMM_HIP_ERR_OVERFLOW, "%s: too many tiles of queries or keys", where);
    *tiles = (int)n;
    return SPMM_HIP_OK;
}

struct WindowKernel { const void *kernel; int rows, threads; };
template <typename T, int DP, int MG, int PG, int SUB> static WindowKernel window_with(bool direct) {
    using S = WindowShape<T, DP, MG, PG, SUB>;
    return {direct ? (const void *)window_kernel<T, DP, MG, PG, SUB, true> : (const void *)window_kernel<T, DP, MG, PG, SUB, false>,
            S::ROWS, S::THREADS};
}
template <typename T, int DP> static WindowKernel window_for(bool direct, bool few) {
    if constexpr (sizeof(T) == 2) return few ? window_with<T, DP, 1, 4, 1>(direct) : window_with<T, DP, 4, 1, 2>(direct);
    else return few ? window_with<T, DP, 1, DP == 64 ? 4 : 2, 1>(direct) : window_with<T, DP, 4, 1, 1>(direct);
}
// few: blocks of the large shape would not fill half of the compute units; blocks of 32 queries then, whose waves share out
// the keys.  512 tokens, 8 heads of 128 in bf16 (32 large blocks): 15.0 us with small blocks, 19.6 with large ones; 2048
// tokens (128): 43.6 and 37.8, 8192 tokens: 186 and 55.  In 32 bits 50 and 89, 198 and 196, 824 and 397.
template <typename T> static WindowKernel window_of(int dim, bool direct, bool few) {
    return dim <= 64 ? window_for<T, 64>(direct, few) : dim <= 96 ? window_for<T, 96>(direct, few) : window_for<T, 128>(direct, few);
}

}  // namespace attn

using namespace attn;

extern "C" int spmm_attn_window(const spmm_attn_desc_t *a, const spmm_attn_rows_t *q, const spmm_attn_rows_t *k,
                                const spmm_attn_rows_t *v, const int32_t *cu_q, const int32_t *cu_k,
                                const spmm_attn_rows_t *out, float *lse, void *stream) {
    const char *W = "attn_window";
    WindowArgs A;
    int st = check_desc(a, W);
    if (st == SPMM_HIP_OK) st = window_args(a, W, cu_q, cu_k, &A);
    if (st != SPMM_HIP_OK) return st;
    const bool packed = cu_q != nullptr;
    const int64_t nb = packed ? 1 : a->batch;
    if ((st = check_rows(a, q, W, "q", nb, a->q_len, a->heads, false, &A.q)) ||
        (st = check_rows(a, k, W, "k", nb, a->k_len, a->kv_heads, false, &A.k)) ||
        (st = check_rows(a, v, W, "v", nb, a->k_len, a->kv_heads, false, &A.v)) ||
        (st = check_rows(a, out, W, "out", nb, a->q_len, a->heads, true, &A.out)))
        return st;
    if (nb == 0 || a->q_len == 0 || (a->batch == 0 && !a->zero_rest)) return SPMM_HIP_OK;      // no sequence: all rows lie behind it
    if (!lse || (uintptr_t)lse % 4) return fail(SPMM_HIP_ERR_ARG, "%s: lse is NULL or not aligned", W);
    A.lse = lse;
    const bool direct = A.k.direct && A.v.direct, few = (nb * a->q_len + 127) / 128 * a->heads < 128;
    const WindowKernel K = a->dtype == SPMM_ATTN_F32 ? window_of<float>(a->dim, direct, few)
                           : a->dtype == SPMM_ATTN_F16 ? window_of<_Float16>(a->dim, direct, few) : window_of<__bf16>(a->dim, direct, few);
    if ((st = tile_count(a, W, packed, a->q_len, K.rows, &A.tiles))) return st;
    OnDevice on(a->device, W);
    if (on.status) return on.status;
    void *args[] = {&A};
    return launch(K.kernel, W, (int64_t)A.tiles * a->heads, K.threads, args, stream);
}
