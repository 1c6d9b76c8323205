// attn_window_grad.hip -- gradients of the window attention (include/spmm_attn.h).
//
// With P = exp(scale Q K^T - lse) on the visible places, D_i = <dO_i, O_i>, dP = dO V^T and dS = P o (dP - D):
//   dV = P^T dO,   dK = scale dS^T Q,   dQ = scale dS K.
// P is formed again from the saved lse instead of being kept.  Two kernels form it, one that owns keys (dK, dV: sums over
// the queries that see them, over every query head of the group in order) and one that owns queries (dQ): seven
// products in place of five, but each sum has one owner, so there are no atomics and no order that varies.
// Layouts as in the forward kernel: a product's result is the next product's operand in registers.
#include "attn_window.hpp"

namespace attn {

// D of 16 rows x heads a block: 16 lanes a row, 8 elements a lane.
template <typename T> __global__ __launch_bounds__(256) void delta_kernel(WindowArgs A) {
    const bool packed = A.cu_q != nullptr;
    const int64_t rows = (packed ? 1 : A.batch) * A.q_len, x = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const bool mine = x < rows * A.heads;
    const int64_t row = mine ? x / A.heads : 0;
    const int head = mine ? (int)(x % A.heads) : 0, e = (threadIdx.x & 15) * 8;
    const int64_t b = packed ? 0 : row / A.q_len, r = packed ? row : row % A.q_len;
    auto at = [&](const Rows &t) { return mine ? (const T *)t.ptr + b * t.seq + r * t.row + head * t.head : nullptr; };
    const frag<T> o = load_frag<T>(at(A.out), e, A.dim, A.out.wide), d = load_frag<T>(at(A.dout), e, A.dim, A.dout.wide);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += (float)o[j] * (float)d[j];
#pragma unroll
    for (int w = 8; w; w /= 2) s += __shfl_xor(s, w);
    if (mine && (threadIdx.x & 15) == 0) A.delta[x] = s;
}

constexpr int GM = 128;                      // rows a workgroup owns, 32 a wave
constexpr int GN = 32;                       // rows of a staged tile

template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void grad_q_kernel(WindowArgs A) {
    using L = Tile<T, DP>;
    constexpr int ND = DP / 32, NS = DP / 16;
    __shared__ __align__(16) T sk[2][GN * L::PITCH];
    __shared__ __align__(16) T sv[2][GN * L::PITCH];
    __shared__ int odd;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    int kv, g, t;
    place(A, A.heads / A.kv_heads, &kv, &g, &t);
    t = A.tiles - 1 - t;
    const int head = kv * (A.heads / A.kv_heads) + g;
    const bool packed = A.cu_q != nullptr;
    const Seq s = find_tile(t, GM, false, A.cu_q, A.cu_k, A.batch, A.q_len, A.k_len);
    if (s.tile < 0) {
        if (A.zero_rest && packed)
            zero_rows<T>(A.dq, s.rest + (int64_t)(t - s.nq) * GM, (int64_t)(A.tiles - s.nq) * GM, GM, A.q_len, head, A.dim);
        return;
    }
    if (tid == 0) odd = 0;
    const int shift = s.nk - s.nq, m0 = s.tile * GM, m1 = min(m0 + GM, s.nq) - 1;
    const int pmin = m0 + shift, pmax = m1 + shift;
    const int lo = A.mask.window ? max(0, pmin - A.mask.window + 1) : 0;
    const int lt = lo / GN, ht = pmax >= 0 ? pmax / GN : -1;
    const int ns = pmax >= 0 ? min((min(A.mask.sinks, pmax + 1) + GN - 1) / GN, lt) : 0;
    const int tiles = ns + max(0, ht - lt + 1);
    auto tile_at = [&](int i) { return (i < ns ? i : lt + i - ns) * GN; };

    const T *kb = seq_base<T>(A.k, s, s.k0, packed, kv), *vb = seq_base<T>(A.v, s, s.k0, packed, kv);
    const int i = m0 + wave * 32 + (lane & 31), p = i + shift;
    const bool mine = i < s.nq;
    const int w0 = m0 + wave * 32 + shift, w1 = min(w0 + 31, pmax);
    frag<T> qf[NS], df[NS];
    float lse2 = INFINITY, delta = 0.f;          // a row that is not there, or sees nothing: exp2(x - inf) = 0
    {
        const T *qr = mine ? seq_base<T>(A.q, s, s.q0, packed, head) + i * A.q.row : nullptr;
        const T *dr = mine ? seq_base<T>(A.dout, s, s.q0, packed, head) + i * A.dout.row : nullptr;
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            qf[st] = load_frag<T>(qr, st * 16 + h * 8, A.dim, A.q.wide);
            df[st] = load_frag<T>(dr, st * 16 + h * 8, A.dim, A.dout.wide);
        }
        if (mine) {
            const int64_t x = (packed ? s.q0 + i : s.b * A.q_len + i) * A.heads + head;
            lse2 = A.lse[x] == -INFINITY ? INFINITY : A.lse[x] * LOG2E;
            delta = A.delta[x];
        }
    }
    using Move = Mover<T, DP, GN, 256>;
    const bool direct = A.k.wide && A.v.wide;
    auto key_row = [&](const T *base, const Rows &R, int j) {
        return j <= pmax && (j >= lo || j < A.mask.sinks) ? base + (int64_t)j * R.row : nullptr;
    };
    auto bring = [&](int j0, int buf, auto how) {
        how(sk[buf], [&](int r) { return key_row(kb, A.k, j0 + r); });
        how(sv[buf], [&](int r) { return key_row(vb, A.v, j0 + r); });
    };
    auto send = [&](T *tile, auto row) { Move::send(tid, A.dim, tile, row); };
    auto copy = [&](T *tile, auto row) { Move::copy(tid, A.dim, tile, row); };
    auto settle = [&](int j0, int buf) {
        if (direct) Move::arrived();
        else bring(j0, buf, copy);
        if (!A.mask.all(pmin, pmax, j0, j0 + GN - 1) && Move::any_not_finite(tid, sk[buf])) odd = 1;
    };
    f32x16 dq[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) dq[d] = zero16();
    __syncthreads();
    if (tiles) {
        if (direct) bring(tile_at(0), 0, send);
        settle(tile_at(0), 0);
    }
    __syncthreads();
    for (int it = 0; it < tiles; ++it) {
        const int j0 = tile_at(it), buf = it & 1;
        if (direct && it + 1 < tiles) bring(tile_at(it + 1), buf ^ 1, send);
        if (w0 <= w1 && A.mask.any(w0, w1, j0, j0 + GN - 1)) {
            const bool full = A.mask.all(w0, w1, j0, j0 + GN - 1);
            f32x16 sc = zero16(), dp = zero16();
#pragma unroll
            for (int st = 0; st < NS; ++st) {
                sc = mma32(L::row_frag(sk[buf], lane & 31, st * 16 + h * 8), qf[st], sc);
                dp = mma32(L::row_frag(sv[buf], lane & 31, st * 16 + h * 8), df[st], dp);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float ds = __builtin_amdgcn_exp2f(sc[r] * A.scale2 - lse2) * (dp[r] - delta);
                sc[r] = full || A.mask.sees(p, j0 + row_of(r) + 4 * h) ? ds : 0.f;
            }
            const bool careful = !full && __builtin_amdgcn_readfirstlane(odd);      // a seen key that is not finite has made the whole row NaN already
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
                const frag<T> dsf = next_operand<T>(sc, k2);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    frag<T> kf = L::col_frag(sk[buf], k2 * 16, d * 32, lane);
                    if (careful) kf = only_finite<T>(kf);
                    dq[d] = mma32(kf, dsf, dq[d]);
                }
            }
        }
        if (it + 1 < tiles) settle(tile_at(it + 1), buf ^ 1);
        __syncthreads();
    }
    if (!mine) return;
    T *dst = seq_base<T>(A.dq, s, s.q0, packed, head) + i * A.dq.row;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            store4<T>(dst, d * 32 + row_of(r) + 4 * h, A.dim, A.dq.wide,
                      f32x4{dq[d][r] * A.scale, dq[d][r + 1] * A.scale, dq[d][r + 2] * A.scale, dq[d][r + 3] * A.scale});
}

template <typename T, int DP>
__global__ __launch_bounds__(256, 1) void grad_kv_kernel(WindowArgs A) {
    using L = Tile<T, DP>;
    constexpr int ND = DP / 32, NS = DP / 16;
    __shared__ __align__(16) T sq[2][GN * L::PITCH];
    __shared__ __align__(16) T sd[2][GN * L::PITCH];
    __shared__ __align__(16) float slse[2][GN], sdelta[2][GN];
    __shared__ int odd;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    int kv, g, t;
    place(A, 1, &kv, &g, &t);
    const bool packed = A.cu_q != nullptr;
    const Seq s = find_tile(t, GM, true, A.cu_q, A.cu_k, A.batch, A.q_len, A.k_len);
    if (s.tile < 0) {
        if (A.zero_rest && packed) {
            const int64_t from = s.rest + (int64_t)(t - s.nq) * GM, step = (int64_t)(A.tiles - s.nq) * GM;
            zero_rows<T>(A.dk, from, step, GM, A.k_len, kv, A.dim);
            zero_rows<T>(A.dv, from, step, GM, A.k_len, kv, A.dim);
        }
        return;
    }
    if (tid == 0) odd = 0;
    const int group = A.heads / A.kv_heads;
    const int shift = s.nk - s.nq, n0 = s.tile * GM, n1 = min(n0 + GM, s.nk) - 1;
    // queries that see some key of the block
    const int i0 = max(0, n0 - shift);
    const int i1 = A.mask.window == 0 || n0 < A.mask.sinks ? s.nq - 1 : min(s.nq - 1, n1 + A.mask.window - 1 - shift);
    const int q0t = i0 / GN, nqt = i1 >= i0 ? i1 / GN - q0t + 1 : 0, tiles = nqt * group;

    const int key = n0 + wave * 32 + (lane & 31);
    const bool mine = key < s.nk;
    const int c0 = n0 + wave * 32, c1 = min(c0 + 31, n1);          // the wave's keys
    frag<T> kf[NS], vf[NS];
    {
        const T *kr = mine ? seq_base<T>(A.k, s, s.k0, packed, kv) + key * A.k.row : nullptr;
        const T *vr = mine ? seq_base<T>(A.v, s, s.k0, packed, kv) + key * A.v.row : nullptr;
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            kf[st] = load_frag<T>(kr, st * 16 + h * 8, A.dim, A.k.wide);
            vf[st] = load_frag<T>(vr, st * 16 + h * 8, A.dim, A.v.wide);
        }
    }
    using Move = Mover<T, DP, GN, 256>;
    const bool direct = A.q.wide && A.dout.wide;
    auto live = [&](int i) { return i >= i0 && i <= i1; };
    auto bring = [&](int it, int buf, auto how) {
        const int head = kv * group + it / nqt, j0 = (q0t + it % nqt) * GN;
        const T *qb = seq_base<T>(A.q, s, s.q0, packed, head), *db = seq_base<T>(A.dout, s, s.q0, packed, head);
        how(sq[buf], [&](int r) { return live(j0 + r) ? qb + (int64_t)(j0 + r) * A.q.row : nullptr; });
        how(sd[buf], [&](int r) { return live(j0 + r) ? db + (int64_t)(j0 + r) * A.dout.row : nullptr; });
    };
    float stat = 0.f;                                // lse or delta of one of the tile's rows, on its way to LDS
    auto load_stat = [&](int it) {
        if (tid >= 2 * GN) return;
        const int head = kv * group + it / nqt, i = (q0t + it % nqt) * GN + tid % GN;
        const int64_t x = ((packed ? s.q0 : s.b * A.q_len) + i) * A.heads + head;
        stat = tid < GN ? INFINITY : 0.f;            // no row, or one that sees nothing: P = exp2(x - inf) = 0
        if (!live(i)) return;
        if (tid >= GN) stat = A.delta[x];
        else if (A.lse[x] != -INFINITY) stat = A.lse[x] * LOG2E;
    };
    auto send = [&](T *tile, auto row) { Move::send(tid, A.dim, tile, row); };
    auto copy = [&](T *tile, auto row) { Move::copy(tid, A.dim, tile, row); };
    auto settle = [&](int it, int buf) {
        const int p0 = (q0t + it % nqt) * GN + shift;
        if (direct) Move::arrived();
        else bring(it, buf, copy);
        if (!A.mask.all(p0, p0 + GN - 1, n0, n1) &&
            (Move::any_not_finite(tid, sq[buf]) || Move::any_not_finite(tid, sd[buf]))) odd = 1;
        if (tid < GN) slse[buf][tid] = stat;
        else if (tid < 2 * GN) sdelta[buf][tid - GN] = stat;
    };
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = zero16();
    __syncthreads();
    if (tiles) {
        load_stat(0);
        if (direct) bring(0, 0, send);
        settle(0, 0);
    }
    __syncthreads();
    for (int it = 0; it < tiles; ++it) {
        const int j0 = (q0t + it % nqt) * GN, p0 = j0 + shift, buf = it & 1;
        if (it + 1 < tiles) {
            load_stat(it + 1);
            if (direct) bring(it + 1, buf ^ 1, send);
        }
        if (c0 <= c1 && A.mask.any(p0, p0 + GN - 1, c0, c1)) {
            const bool full = A.mask.all(p0, p0 + GN - 1, c0, c1);
            f32x16 sc = zero16(), dp = zero16();
#pragma unroll
            for (int st = 0; st < NS; ++st) {
                sc = mma32(L::row_frag(sq[buf], lane & 31, st * 16 + h * 8), kf[st], sc);
                dp = mma32(L::row_frag(sd[buf], lane & 31, st * 16 + h * 8), vf[st], dp);
            }
#pragma unroll
            for (int r4 = 0; r4 < 16; r4 += 4) {
                const f32x4 l4 = *reinterpret_cast<const f32x4 *>(&slse[buf][row_of(r4) + 4 * h]);
                const f32x4 d4 = *reinterpret_cast<const f32x4 *>(&sdelta[buf][row_of(r4) + 4 * h]);
#pragma unroll
                for (int r = r4; r < r4 + 4; ++r) {
                    const bool seen = full || A.mask.sees(p0 + row_of(r) + 4 * h, key);
                    const float pr = __builtin_amdgcn_exp2f(sc[r] * A.scale2 - l4[r - r4]);
                    dp[r] = seen ? pr * (dp[r] - d4[r - r4]) : 0.f;
                    sc[r] = seen ? pr : 0.f;
                }
            }
            const bool careful = !full && __builtin_amdgcn_readfirstlane(odd);
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
                const frag<T> pf = next_operand<T>(sc, k2), dsf = next_operand<T>(dp, k2);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    frag<T> of = L::col_frag(sd[buf], k2 * 16, d * 32, lane), qf = L::col_frag(sq[buf], k2 * 16, d * 32, lane);
                    if (careful) {
                        of = only_finite<T>(of);
                        qf = only_finite<T>(qf);     // a query that is not finite has an lse that is not, so NaN in dsf
                    }
                    dv[d] = mma32(of, pf, dv[d]);
                    dk[d] = mma32(qf, dsf, dk[d]);
                }
            }
            if (careful)
                add_not_finite<T, DP>(dv, sd[buf], GN, lane, [&](int r) { return j0 + r <= i1 && A.mask.sees(p0 + r, key); });
        }
        if (it + 1 < tiles) settle(it + 1, buf ^ 1);
        __syncthreads();
    }
    if (!mine) return;
    T *kd = seq_base<T>(A.dk, s, s.k0, packed, kv) + key * A.dk.row, *vd = seq_base<T>(A.dv, s, s.k0, packed, kv) + key * A.dv.row;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            store4<T>(kd, d * 32 + row_of(r) + 4 * h, A.dim, A.dk.wide,
                      f32x4{dk[d][r] * A.scale, dk[d][r + 1] * A.scale, dk[d][r + 2] * A.scale, dk[d][r + 3] * A.scale});
            store4<T>(vd, d * 32 + row_of(r) + 4 * h, A.dim, A.dv.wide,
                      f32x4{dv[d][r], dv[d][r + 1], dv[d][r + 2], dv[d][r + 3]});
        }
}

struct GradKernels { const void *delta, *q, *kv; };
template <typename T> static GradKernels grads_of(int dim) {
    const void *d = (const void *)delta_kernel<T>;
    if (dim <= 64) return {d, (const void *)grad_q_kernel<T, 64>, (const void *)grad_kv_kernel<T, 64>};
    if (dim <= 96) return {d, (const void *)grad_q_kernel<T, 96>, (const void *)grad_kv_kernel<T, 96>};
    return {d, (const void *)grad_q_kernel<T, 128>, (const void *)grad_kv_kernel<T, 128>};
}

}  // namespace attn

using namespace attn;

extern "C" int spmm_attn_window_work(const spmm_attn_desc_t *a, int32_t packed, size_t *bytes) {
    const int st = check_desc(a, "attn_window_work");
    if (st != SPMM_HIP_OK) return st;
    if (!bytes) return fail(SPMM_HIP_ERR_ARG, "attn_window_work: bytes is NULL");
    const int64_t n = packed ? 1 : a->batch;
    if (n && a->q_len > (INT64_C(1) << 44) / n / a->heads) return fail(SPMM_HIP_ERR_OVERFLOW, "attn_window_work: too many rows");
    *bytes = (size_t)(n * a->q_len * a->heads) * 4;
    return SPMM_HIP_OK;
}

extern "C" int spmm_attn_window_grad(const spmm_attn_desc_t *a, const spmm_attn_rows_t *dout, const spmm_attn_rows_t *q,
                                     const spmm_attn_rows_t *k, const spmm_attn_rows_t *v, const spmm_attn_rows_t *out,
                                     const float *lse, const int32_t *cu_q, const int32_t *cu_k,
                                     const spmm_attn_rows_t *dq, const spmm_attn_rows_t *dk, const spmm_attn_rows_t *dv,
                                     void *work, size_t work_bytes, void *stream) {
    const char *W = "attn_window_grad";
    WindowArgs A;
    int st = check_desc(a, W);
    if (st == SPMM_HIP_OK) st = window_args(a, W, cu_q, cu_k, &A);
    if (st != SPMM_HIP_OK) return st;
    const bool packed = cu_q != nullptr;
    const int64_t nb = packed ? 1 : a->batch;
    if ((st = check_rows(a, dout, W, "dout", nb, a->q_len, a->heads, false, &A.dout)) ||
        (st = check_rows(a, q, W, "q", nb, a->q_len, a->heads, false, &A.q)) ||
        (st = check_rows(a, k, W, "k", nb, a->k_len, a->kv_heads, false, &A.k)) ||
        (st = check_rows(a, v, W, "v", nb, a->k_len, a->kv_heads, false, &A.v)) ||
        (st = check_rows(a, out, W, "out", nb, a->q_len, a->heads, false, &A.out)) ||
        (st = check_rows(a, dq, W, "dq", nb, a->q_len, a->heads, true, &A.dq)) ||
        (st = check_rows(a, dk, W, "dk", nb, a->k_len, a->kv_heads, true, &A.dk)) ||
        (st = check_rows(a, dv, W, "dv", nb, a->k_len, a->kv_heads, true, &A.dv)))
        return st;
    if (a->batch == 0) return SPMM_HIP_OK;
    size_t need = 0;
    if ((st = spmm_attn_window_work(a, packed, &need))) return st;
    if (need > 0) {
        if (!lse || (uintptr_t)lse % 4) return fail(SPMM_HIP_ERR_ARG, "%s: lse is NULL or not aligned", W);
        if (!work || (uintptr_t)work % 16 || work_bytes < need)
            return fail(SPMM_HIP_ERR_ARG, "%s: the workspace needs %zu bytes, 16-byte aligned", W, need);
    }
    A.lse = const_cast<float *>(lse);
    A.delta = (float *)work;
    int qt = 0, kt = 0;
    if (a->q_len > 0 && (st = tile_count(a, W, packed, a->q_len, GM, &qt))) return st;
    if (a->k_len > 0 && (st = tile_count(a, W, packed, a->k_len, GM, &kt))) return st;
    OnDevice on(a->device, W);
    if (on.status) return on.status;
    const GradKernels G = a->dtype == SPMM_ATTN_F32 ? grads_of<float>(a->dim)
                          : a->dtype == SPMM_ATTN_F16 ? grads_of<_Float16>(a->dim) : grads_of<__bf16>(a->dim);
    void *args[] = {&A};
    const int64_t rows = nb * a->q_len * a->heads;
    if ((st = launch(G.delta, W, (rows + 15) / 16, 256, args, stream))) return st;
    A.tiles = kt;
    if ((st = launch(G.kv, W, (int64_t)kt * a->kv_heads, 256, args, stream))) return st;
    A.tiles = qt;
    return launch(G.q, W, (int64_t)qt * a->heads, 256, args, stream);
}
