// attn_window_grad.hip -- gradients of the window attention (include/spmm_attn.h).
//
// With P = exp(scale Q K^T - lse) on the visible places, D_i = <dO_i, O_i>, dP = dO V^T and dS = P o (dP - D):
//   dV = P^T dO,   dK = scale dS^T Q,   dQ = scale dS K.
// P is formed again from the saved lse instead of being kept.  Two kernels form it, one that owns queries (dQ) and one that
// owns keys (dK, dV: sums over the queries that see them, over every query head of the group in order): seven
// products in place of five, but each sum has one owner, so there are no atomics and no order that varies.
// With 16-bit types P and dS are rounded to them for dV and dK.  For dQ dS goes in two 16-bit parts, and the row sum of dS,
// which is zero but for the rounding of out in D, corrects D for dK.  Both are held as multiples that float16 has normal
// numbers for (Lift, Factor).
// Layouts as in the forward kernel: a product's result is the next product's operand in registers.
//
// Bound: matrix instructions, exponentials and the reads of LDS that feed them.  Two sequences of 8192 and 8000 tokens, 32
// heads over 8 of 128 in bf16, window 1024, 4 first keys: 1720 to 1775 us with the forward pass, 505 to 520 TFLOP/s of the seven
// products that the formulas need, of ten that are made.  In a trace, which slows them by a tenth, the means are delta 53 us
// (the bytes of out and dout), grad_q 625, grad_kv 827, join 17, forward 407; matrix units busy for 46 (grad_q) and 34 %
// (grad_kv) of the cycles, vector units for 46 and 29, LDS for 18 and 27.  Keeping V's fragments in registers as well, or two
// half tiles in turn, spills and is slower (2455 and 2300 us).
//
// 257 tokens, 4 heads over 2 of 64 in 32 bits: grad_kv 39 us, grad_q 21, forward 19, join 5, delta 4, in all 84: eighteen blocks of
// keys and a few more on 256 compute units, each of which walks its tiles in turn.
#include "attn_window.hpp"

namespace attn {

// float16 has normal numbers from 2^-14 to 2^16, and P over thousands of keys, or dS for an ordinary gradient of 1e-4, lies
// below them.  P, which is 1 at most, is formed as 2^P times itself: the row's lse is smaller by P in the exponent.
template <typename T> struct Lift { static constexpr int P = 0; };
template <> struct Lift<_Float16> { static constexpr int P = 12; };

// And dS enters its products times a power of two for each sum, a lane's column: the largest |dS| met so far is at 2^7 or more
// times it, at 2^15 at most.  What is 2^-21 of that or more keeps all its bits, the rest is off by 2^-32 of it.  Sums so far
// are brought to the new factor when it falls, which is rare, and all of it is exact.  Maximum, test and product make the
// gradients of 4096 tokens, 8 heads over 2 of 128, window 1024 in fp16 190 us from 178, of 8192 tokens, 32 heads over 8, 824
// from 777.  The other types have exponents enough.
template <typename T> struct Factor {
    static constexpr bool USED = Lift<T>::P > 0;
    float f = USED ? 0x1p100f : 1.f;

    template <int ND> __device__ __forceinline__ void apply(f32x16 &x, f32x16 (&acc)[ND]) {
        if constexpr (USED) {
            float top = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(x[r]));
            top = fmaxf(top, __shfl_xor(top, 32));
            const bool over = top * f > 0x1p15f;
            if (__any(over)) {
                // 2^7 over the maximum's power of two; above 2^-85 it is, so its exponent is 42 or more
                const float g = over ? __builtin_bit_cast(float, (261u - (__builtin_bit_cast(uint32_t, top) >> 23)) << 23) : f;
                const float by = g * (1.f / f);
#pragma unroll
                for (int d = 0; d < ND; ++d) acc[d] *= by;
                f = g;
            }
            x *= f;
        }
    }
    // the sums as they are, of P or dS times 2^P
    template <int ND> __device__ __forceinline__ void remove(f32x16 (&acc)[ND]) const {
        if constexpr (USED) {
            const float by = 1.f / f * (1.f / (1 << Lift<T>::P));
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[d] *= by;
        }
    }
};

// What the two kernels below need of every query row, 16 rows x heads a block, 16 lanes a row, 8 elements a lane:
// lse in powers of two, less Lift::P (+inf where the query sees nothing: every weight is then exp2(x - inf) = 0), and -D.
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
    if (mine && (threadIdx.x & 15) == 0) {
        const float l = A.lse[x];
        A.stats[2 * x] = l == -INFINITY ? INFINITY : l * LOG2E - Lift<T>::P;
        A.stats[2 * x + 1] = -s;
    }
}

// How a block is made up: as in the forward kernel, MG groups of 32 queries times PG waves that share a group's keys, 32 SUB
// of every tile each.
template <typename T, int DP, int MG, int PG, int SUB> struct QShape {
    static constexpr int ROWS = 32 * MG, KN = 32 * PG * SUB, THREADS = 64 * MG * PG;
};

template <typename T, int DP, int MG, int PG, int SUB, bool DIRECT>
__global__ __launch_bounds__(64 * MG * PG, sizeof(T) == 2 && PG == 1 ? 2 : 1) void grad_q_kernel(WindowArgs A) {
    using L = Tile<T, DP>;
    using S = QShape<T, DP, MG, PG, SUB>;
    constexpr int GM = S::ROWS, GN = S::KN, THREADS = S::THREADS, ND = DP / 32, NS = DP / 16;
    __shared__ __align__(16) T sk[2][GN * L::PITCH], sv[2][GN * L::PITCH];
    __shared__ int odd[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5;
    const int mg = wave % MG, part = wave / MG;      // the wave's queries, and which keys of a tile
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
    if (tid == 0) odd[0] = odd[1] = 0;
    const int shift = s.nk - s.nq, m0 = s.tile * GM, m1 = min(m0 + GM, s.nq) - 1;
    const int pmin = m0 + shift, pmax = m1 + shift;
    const int lo = A.mask.window ? max(0, pmin - A.mask.window + 1) : 0;
    const int lt = lo / GN, ht = pmax >= 0 ? pmax / GN : -1;
    const int ns = pmax >= 0 ? min((min(A.mask.sinks, pmax + 1) + GN - 1) / GN, lt) : 0;
    const int tiles = ns + max(0, ht - lt + 1);
    auto tile_at = [&](int i) { return (i < ns ? i : lt + i - ns) * GN; };

    const T *kb = seq_base<T>(A.k, s, s.k0, packed, kv), *vb = seq_base<T>(A.v, s, s.k0, packed, kv);
    const int i = m0 + mg * 32 + (lane & 31), p = i + shift;
    const bool mine = i < s.nq;
    const int w0 = m0 + mg * 32 + shift, w1 = min(w0 + 31, pmax);
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
        settled<T>(qf);
        settled<T>(df);
        if (mine) {
            const int64_t x = (packed ? s.q0 + i : s.b * A.q_len + i) * A.heads + head;
            lse2 = A.stats[2 * x];
            delta = A.stats[2 * x + 1];
        }
        asm volatile("" : "+v"(lse2), "+v"(delta));
    }
    using Move = Mover<T, DP, GN, THREADS>;
    Move mk, mv;
    if (DIRECT) {
        mk.start(tid, A.dim, A.k.row);
        mv.start(tid, A.dim, A.v.row);
    }
    auto send = [&](int j0, T *tk, T *tv) {
        mk.send(wave, tk, kb + (int64_t)j0 * A.k.row, A.k.row, pmax + 1 - j0, A.dim);
        mv.send(wave, tv, vb + (int64_t)j0 * A.v.row, A.v.row, pmax + 1 - j0, A.dim);
    };
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
        if (!A.mask.all(pmin, pmax, j0, j0 + GN - 1) && Move::any_not_finite(tid, tk)) odd[buf] = 1;
    };
    f32x16 dq[ND];
    float left;                                      // sum of the row's 2^P dS
    Factor<T> factor;
    auto step = [&](auto careful, int j0, const T *tk, const T *tv) __attribute__((always_inline)) {
        const bool full = A.mask.all(w0, w1, j0, j0 + 31);
        f32x16 sc = zero16(), dp;                    // dP - D: the sums start from -D
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] = delta;
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            sc = mma32(L::row_frag(tk, lane & 31, st * 16 + h * 8), qf[st], sc);
            dp = mma32(L::row_frag(tv, lane & 31, st * 16 + h * 8), df[st], dp);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r)
            sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], A.scale2, -lse2)) * dp[r];
        if (!full) {
            asm volatile("");                        // a branch, not 16 selects in every tile
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (!A.mask.sees(p, j0 + row_of(r) + 4 * h)) sc[r] = 0.f;
        }
        // a seen key that is not finite makes the row's weights NaN, so it need not be put back
#pragma unroll
        for (int r = 0; r < 16; ++r) left += sc[r];
        factor.apply(sc, dq);
        if constexpr (!careful) {
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
                const frag<T> dsf = next_operand<T>(sc, k2);
                frag<T> low = {};                    // what rounding dS to 16 bits leaves
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) low[j] = narrow<T>(sc[8 * k2 + j] - (float)dsf[j]);
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const frag<T> kf = L::col_frag(tk, k2 * 16, d * 32, lane);
                    dq[d] = mma32(kf, dsf, dq[d]);
                    if constexpr (sizeof(T) == 2) dq[d] = mma32(kf, low, dq[d]);
                }
            }
        } else {
            Careful<T, DP, 32> c;
            for (int d = 0; d < ND; ++d) c.acc[d] = dq[d];
            c.w[0] = sc;
            careful_product<T, DP, 32, sizeof(T) == 2>(&c, tk, lane, A.mask, p, j0, true, -1);
            for (int d = 0; d < ND; ++d) dq[d] = c.acc[d];
        }
    };
    // as in the forward kernel: false if a value in a partly seen tile is not finite
    auto run = [&](auto careful) {
#pragma unroll
        for (int d = 0; d < ND; ++d) dq[d] = zero16();
        left = 0.f;
        factor = {};
        if (tiles) {
            if (DIRECT) send(tile_at(0), sk[0], sv[0]);
            settle(tile_at(0), 0, sk[0], sv[0]);
        }
        __syncthreads();
        for (int it = 0; it < tiles; ++it) {
            const int buf = it & 1, j0 = tile_at(it);
            if (!careful && !A.mask.all(pmin, pmax, j0, j0 + GN - 1) && uniform(odd[buf])) return false;
            const bool more = it + 1 < tiles;
            if (DIRECT && more) send(tile_at(it + 1), sk[buf ^ 1], sv[buf ^ 1]);
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const int r = 32 * (SUB * part + u);
                step(careful, j0 + r, sk[buf] + r * L::PITCH, sv[buf] + r * L::PITCH);
            }
            if (more) settle(tile_at(it + 1), buf ^ 1, sk[buf ^ 1], sv[buf ^ 1]);
            __syncthreads();
        }
        return true;
    };
    __syncthreads();
    if (!run(std::false_type{})) {
        __syncthreads();
        run(std::true_type{});
    }
    factor.remove(dq);
    left += __shfl_xor(left, 32);
    left *= 1.f / (1 << Lift<T>::P);
    if constexpr (PG > 1) {                          // the parts' sums, in order, through the tiles' place in LDS
        float *mail = reinterpret_cast<float *>(sk) + mg * ND * 16 * 64 + lane;
#pragma unroll 1
        for (int from = 1; from < PG; ++from) {
            if (from > 1) __syncthreads();
            if (part == from) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) mail[(d * 16 + r) * 64] = dq[d][r];
                mail[ND * 16 * 64 * MG] = left;
            }
            __syncthreads();
            if (part == 0) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) dq[d][r] += mail[(d * 16 + r) * 64];
                left += mail[ND * 16 * 64 * MG];
            }
        }
    }
    if (!mine || part != 0) return;
    // A row of dS sums to zero; what is left is by how much D, taken from the rounded out, is off.  The kernel that owns keys
    // runs next and gets it right.
    if (h == 0) A.stats[2 * ((packed ? s.q0 + i : s.b * A.q_len + i) * A.heads + head) + 1] -= left;
    T *dst = seq_base<T>(A.dq, s, s.q0, packed, head) + i * A.dq.row;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            store4<T>(dst, d * 32 + row_of(r) + 4 * h, A.dim, A.dq.wide,
                      f32x4{dq[d][r] * A.scale, dq[d][r + 1] * A.scale, dq[d][r + 2] * A.scale, dq[d][r + 3] * A.scale});
}

// The first keys that stay visible are seen by every later query, the others by a window of them: were their block to
// take all its queries, it would be many times the others' length and the last to end.  So with few of them (A.chunk > 0)
// their block takes its window's queries only, further blocks take chunks of the other queries each, and what
// they find for these keys goes to `part` in 32 bits and is summed in order by join_kernel.
__device__ __forceinline__ float *part_of(const WindowArgs &A, int64_t slot, int kv) {
    return A.part + (slot * A.kv_heads + kv) * 2 * A.mask.sinks * A.dim;
}
__device__ __forceinline__ int64_t chunk_slot(const WindowArgs &A, const Seq &s, bool packed, int c) {
    return A.batch + (packed ? s.q0 / A.chunk + s.b : s.b * ((A.q_len + A.chunk - 1) / A.chunk)) + c;
}
// last query that sees one of the keys n0 .. n1 through the window
__device__ __forceinline__ int window_end(const WindowArgs &A, const Seq &s, int n1) {
    return (int)min((int64_t)s.nq - 1, (int64_t)n1 + A.mask.window - 1 - (s.nk - s.nq));
}

// How a block of the kernel below is made up: KG groups of 32 keys, whose keys and values stay in LDS, times PG waves that
// share a group's queries, 32 of every tile each, and add up in order at the end; STAGES tiles of 32 PG queries on
// their way or in use.
template <typename T, int DP, int KG, int PG> struct KvShape {
    static constexpr int KEYS = 32 * KG, QN = 32 * PG, THREADS = 64 * KG * PG;
    static constexpr int TILE = 2 * QN * Tile<T, DP>::PITCH * (int)sizeof(T) + 8 * QN;
    static constexpr int KV = 2 * KEYS * Tile<T, DP>::PITCH * (int)sizeof(T);
    static constexpr int STAGES = (160 * 1024 - 64 - KV) / TILE < 4 ? (160 * 1024 - 64 - KV) / TILE : 4;
    static_assert(STAGES >= 1, "one tile has to fit");
};
template <typename T, int DP, int KG, int PG> struct KvShared {
    using S = KvShape<T, DP, KG, PG>;
    static constexpr int P = Tile<T, DP>::PITCH;
    __align__(16) T k[S::KEYS * P], v[S::KEYS * P];                  // at the end: a wave's sums for another
    __align__(16) T q[S::STAGES][S::QN * P], d[S::STAGES][S::QN * P];
    __align__(16) float s[S::STAGES][2 * S::QN];                     // lse and D of the tile's rows
    int odd[2];                                                      // a value of tile 0, 2, .. or 1, 3, .. is not finite
};

// False, with nothing written, if a value in a partly seen tile is not finite and CAREFUL does not allow for that.
template <typename T, int DP, int KG, int PG, bool DIRECT, bool CAREFUL>
__device__ __forceinline__ bool grad_kv_block(const WindowArgs &A, KvShared<T, DP, KG, PG> &sh) {
    using L = Tile<T, DP>;
    using S = KvShape<T, DP, KG, PG>;
    constexpr int ND = DP / 32, NS = DP / 16, QN = S::QN, KEYS = S::KEYS, STAGES = S::STAGES, THREADS = S::THREADS;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5;
    const int kg = wave % KG, part = wave / KG;                       // the wave's keys, and which queries of a tile
    // the blocks that own keys, then those that take a chunk of queries for a block of the first keys each
    const int ke = (A.mask.sinks + KEYS - 1) / KEYS;
    int t = (int)blockIdx.x, e0 = 0;
    const bool packed = A.cu_q != nullptr, extra = t >= A.tiles * A.kv_heads;
    if (extra) t -= A.tiles * A.kv_heads;
    const int kv = t % A.kv_heads;
    t /= A.kv_heads;
    if (extra) {
        e0 = t % ke;
        t /= ke;
    }
    const Seq s = extra ? find_tile(t, A.chunk, false, A.cu_q, A.cu_k, A.batch, A.q_len, A.k_len)
                        : find_tile(t, KEYS, true, A.cu_q, A.cu_k, A.batch, A.q_len, A.k_len);
    if (s.tile < 0) {
        if (A.zero_rest && packed && !extra) {
            const int64_t from = s.rest + (int64_t)(t - s.nq) * KEYS, step = (int64_t)(A.tiles - s.nq) * KEYS;
            zero_rows<T>(A.dk, from, step, KEYS, A.k_len, kv, A.dim);
            zero_rows<T>(A.dv, from, step, KEYS, A.k_len, kv, A.dim);
        }
        return true;
    }
    if (tid == 0) sh.odd[0] = sh.odd[1] = 0;
    const int group = A.heads / A.kv_heads;
    const int shift = s.nk - s.nq, n0 = (extra ? e0 : s.tile) * KEYS;
    const int n1 = min(n0 + KEYS, extra ? min(A.mask.sinks, s.nk) : s.nk) - 1;
    const bool first = A.chunk > 0 && n0 < A.mask.sinks;            // the first keys' results go to `part`
    // queries that see some key of the block
    int i0 = max(0, n0 - shift);
    int i1 = A.mask.window == 0 || (n0 < A.mask.sinks && !first) ? s.nq - 1 : window_end(A, s, n1);
    if (extra) {
        i0 = max(s.tile * A.chunk, window_end(A, s, min(n0 + KEYS, s.nk) - 1) + 1);
        i1 = min((s.tile + 1) * A.chunk, s.nq) - 1;
        if (i1 < i0 || n1 < n0) return true;
    }
    const int first_j = i0 / QN * QN, per_head = i1 >= i0 ? (i1 - first_j) / QN + 1 : 0, tiles = per_head * group;

    const int key = n0 + kg * 32 + (lane & 31);
    const bool mine = key <= n1;
    const T *kb = seq_base<T>(A.k, s, s.k0, packed, kv) + n0 * A.k.row, *vb = seq_base<T>(A.v, s, s.k0, packed, kv) + n0 * A.v.row;
    using MoveK = Mover<T, DP, KEYS, THREADS>;
    using Move = Mover<T, DP, QN, THREADS>;
    constexpr int LOADS = 2 * Move::N + 1;                           // of a tile, a wave
    Move mq, md;
    if (DIRECT) {
        MoveK mk;
        mk.start(tid, A.dim, A.k.row);
        mk.send(wave, sh.k, kb, A.k.row, n1 + 1 - n0, A.dim);
        mk.start(tid, A.dim, A.v.row);
        mk.send(wave, sh.v, vb, A.v.row, n1 + 1 - n0, A.dim);
        mq.start(tid, A.dim, A.q.row);
        md.start(tid, A.dim, A.dout.row);
    } else {
        MoveK::copy(tid, A.dim, sh.k, [&](int r) { return n0 + r <= n1 ? kb + r * A.k.row : nullptr; });
        MoveK::copy(tid, A.dim, sh.v, [&](int r) { return n0 + r <= n1 ? vb + r * A.v.row : nullptr; });
    }
    // The tile that is fetched next: the group's heads one after the other, the queries of each from first_j on.  Past the
    // last there are no rows.
    int next_left = tiles, next_j = first_j, next_g = 0;
    const T *next_q = nullptr, *next_d = nullptr;
    const float *next_s = nullptr;
    auto rewind = [&] {
        const int head = kv * group + next_g;
        next_j = first_j;
        next_q = seq_base<T>(A.q, s, s.q0, packed, head) + (int64_t)first_j * A.q.row;
        next_d = seq_base<T>(A.dout, s, s.q0, packed, head) + (int64_t)first_j * A.dout.row;
        next_s = A.stats + (((packed ? s.q0 : s.b * A.q_len) + first_j) * A.heads + head) * 2;
    };
    if (tiles) rewind();
    auto advance = [&]() __attribute__((always_inline)) {
        next_q += QN * A.q.row;
        next_d += QN * A.dout.row;
        next_s += (int64_t)QN * A.heads * 2;
        next_j += QN;
        --next_left;
        if (next_j > i1 && next_left > 0) {
            ++next_g;
            rewind();
        }
    };
    auto fetch = [&](int buf) __attribute__((always_inline)) {
        const int rows = next_left > 0 ? s.nq - next_j : 0;
        if constexpr (DIRECT) {
            mq.send(wave, sh.q[buf], next_q, A.q.row, rows, A.dim);
            md.send(wave, sh.d[buf], next_d, A.dout.row, rows, A.dim);
            // the rows of this wave's queries: every wave the same number of loads
            const int n = max(0, min(rows - 32 * part, 32));
            const Buffer b(next_s + (int64_t)32 * part * A.heads * 2, n > 0 ? ((n - 1) * A.heads + 1) * 8 : 0);
            b.to_lds4(sh.s[buf] + 64 * part, (lane & 31) * A.heads * 8 + h * 4);      // 32 lse, then 32 -D
        } else {
            Move::copy(tid, A.dim, sh.q[buf], [&](int r) { return r < rows ? next_q + r * A.q.row : nullptr; });
            Move::copy(tid, A.dim, sh.d[buf], [&](int r) { return r < rows ? next_d + r * A.dout.row : nullptr; });
            for (int e = tid; e < 2 * QN; e += THREADS) {
                const int r = e / 64 * 32 + e % 32;
                sh.s[buf][e] = r < rows ? next_s[(int64_t)r * A.heads * 2 + e / 32 % 2] : 0.f;
            }
        }
        advance();
    };
    f32x16 dk[ND], dv[ND];
    Factor<T> factor;                                // of dS
    // the positions plo .. plo + seen - 1 are those of the block's queries that see this lane's key
    const int plo = max(key, i0 + shift);
    const int phi = min(i1 + shift, A.mask.window == 0 || key < A.mask.sinks ? INT32_MAX : key + A.mask.window - 1);
    const unsigned seen = (unsigned)max(0, phi - plo + 1);
    // tiles that start in [all_a, all_b] are seen by every key of the block, the wave's 32 queries that start in [own_a, own_b]
    // by every key of the wave
    const int c0 = n0 + kg * 32, c1 = min(c0 + 31, n1);
    auto last_for = [&](int a, int b) { return A.mask.window == 0 || b < A.mask.sinks ? i1 : min(i1, a + A.mask.window - 1 - shift); };
    const int all_a = max(n1 - shift, i0), all_b = last_for(n0, n1) - QN + 1;
    const int own_a = max(c1 - shift, i0), own_b = last_for(c0, c1) - 31;
    frag<T> kf[sizeof(T) == 2 ? NS : 1];             // the wave's keys: 32-bit ones would take twice the registers
    // rows behind the last query are zeros, what is kept of their lse and D too: 2^P P = 1 then, and adds 1 * 0
    auto step = [&](int j0, const T *tq, const T *td, const float *ts) __attribute__((always_inline)) {
        f32x16 sc = zero16(), dp;                    // dP - D: the sums start from -D
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(ts + 32 + row_of(r) + 4 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) dp[r + i] = x[i];
        }
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            const frag<T> k = sizeof(T) == 2 ? kf[st % (sizeof(T) == 2 ? NS : 1)] : L::row_frag(sh.k, kg * 32 + (lane & 31), st * 16 + h * 8);
            sc = mma32(L::row_frag(tq, lane & 31, st * 16 + h * 8), k, sc);
            dp = mma32(L::row_frag(td, lane & 31, st * 16 + h * 8), L::row_frag(sh.v, kg * 32 + (lane & 31), st * 16 + h * 8), dp);
        }
#pragma unroll
        for (int r4 = 0; r4 < 16; r4 += 4) {
            const f32x4 l = *reinterpret_cast<const f32x4 *>(ts + row_of(r4) + 4 * h);
#pragma unroll
            for (int r = r4; r < r4 + 4; ++r) {
                sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], A.scale2, -l[r - r4]));
                dp[r] = sc[r] * dp[r];
            }
        }
        if (j0 < own_a || j0 > own_b) {
            asm volatile("");                        // a branch, not 16 selects in every tile
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if ((unsigned)(j0 + shift + row_of(r) + 4 * h - plo) >= seen) sc[r] = dp[r] = 0.f;
        }
        factor.apply(dp, dk);
        if constexpr (!CAREFUL) {
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
                const frag<T> pf = next_operand<T>(sc, k2), dsf = next_operand<T>(dp, k2);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    dv[d] = mma32(L::col_frag(td, k2 * 16, d * 32, lane), pf, dv[d]);
                    dk[d] = mma32(L::col_frag(tq, k2 * 16, d * 32, lane), dsf, dk[d]);
                }
            }
        } else {
            // a query that is not finite has an lse that is not, so its weights are NaN: it need not be put back
            Careful<T, DP, 32> c;
            for (int d = 0; d < ND; ++d) c.acc[d] = dv[d];
            c.w[0] = sc;
            careful_product<T, DP, 32>(&c, td, lane, A.mask, key, j0 + shift, false, i1 + shift);
            for (int d = 0; d < ND; ++d) dv[d] = c.acc[d];
            for (int d = 0; d < ND; ++d) c.acc[d] = dk[d];
            c.w[0] = dp;
            careful_product<T, DP, 32>(&c, tq, lane, A.mask, key, j0 + shift, false, INT32_MIN);
            for (int d = 0; d < ND; ++d) dk[d] = c.acc[d];
        }
    };
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = zero16();
    constexpr bool AHEAD = DIRECT && STAGES > 1;
    if (DIRECT) {
        arrived();                                   // keys and values
        if (AHEAD) {
#pragma unroll
            for (int it = 0; it < STAGES - 1; ++it) fetch(it);
        }
    }
    __syncthreads();
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int st = 0; st < NS; ++st) kf[st] = L::row_frag(sh.k, kg * 32 + (lane & 31), st * 16 + h * 8);
        settled<T>(kf);
    }
    bool fine = true;
    for (int it = 0, j0 = first_j, buf = 0; it < tiles; ++it) {
        if (AHEAD) {
            arrived<(STAGES - 2) * LOADS>();
        } else {
            fetch(buf);
            if (DIRECT) arrived();
        }
        const bool whole = j0 >= all_a && j0 <= all_b;
        if (!whole && (Move::any_not_finite(tid, sh.q[buf]) || Move::any_not_finite(tid, sh.d[buf]))) sh.odd[it & 1] = 1;
        __syncthreads();                             // tile `it` is there for all, and tile `it` - 1 is read
        // the whole block leaves at the same tile: what a wave ahead finds in the next one goes to the other flag
        if (!CAREFUL && !whole && uniform(sh.odd[it & 1])) {
            fine = false;
            break;
        }
        if (AHEAD) fetch(buf == 0 ? STAGES - 1 : buf - 1);
        step(j0 + 32 * part, sh.q[buf] + 32 * part * L::PITCH, sh.d[buf] + 32 * part * L::PITCH, sh.s[buf] + 64 * part);
        if (!AHEAD) __syncthreads();
        if (AHEAD) buf = buf == STAGES - 1 ? 0 : buf + 1;
        j0 += QN;
        if (j0 > i1) j0 = first_j;
    }
    if (DIRECT) arrived();
    if (!fine) return false;
    factor.remove(dk);
    Factor<T>{1.f}.remove(dv);
    if constexpr (PG > 1) {                          // the parts' sums, in order, through the keys' place in LDS
        float *mail = reinterpret_cast<float *>(sh.k) + kg * ND * 16 * 64 + lane;
        auto pass = [&](f32x16 (&x)[ND]) {
#pragma unroll 1
            for (int from = 1; from < PG; ++from) {
                __syncthreads();
                if (part == from) {
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int r = 0; r < 16; ++r) mail[(d * 16 + r) * 64] = x[d][r];
                }
                __syncthreads();
                if (part == 0) {
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int r = 0; r < 16; ++r) x[d][r] += mail[(d * 16 + r) * 64];
                }
            }
        };
        pass(dk);
        pass(dv);
    }
    if (!mine || part != 0) return true;
    if (first && key < A.mask.sinks) {
        float *pk = part_of(A, extra ? chunk_slot(A, s, packed, s.tile) : s.b, kv) + key * A.dim, *pv = pk + A.mask.sinks * A.dim;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int e = d * 32 + row_of(r) + 4 * h;
                if (e < A.dim) {
                    pk[e] = dk[d][r];
                    pv[e] = dv[d][r];
                }
            }
        return true;
    }
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
    return true;
}
// The rare case in a function of its own, which takes no registers from the loop above.
template <typename T, int DP, int KG, int PG>
__device__ __attribute__((noinline)) void grad_kv_again(const WindowArgs *A, KvShared<T, DP, KG, PG> *sh) {
    grad_kv_block<T, DP, KG, PG, false, true>(*A, *sh);
}
template <typename T, int DP, int KG, int PG, bool DIRECT>
__global__ __launch_bounds__(64 * KG * PG, KG * PG == 8 ? 2 : 1) void grad_kv_kernel(WindowArgs A) {
    __shared__ KvShared<T, DP, KG, PG> sh;
    if (!grad_kv_block<T, DP, KG, PG, DIRECT, false>(A, sh)) {
        __syncthreads();
        const WindowArgs copy = A;
        grad_kv_again<T, DP, KG, PG>(&copy, &sh);
    }
}

// One wave a (sequence, key head, first key): the window's part and the chunks' parts, in order.
template <typename T> __global__ __launch_bounds__(64) void join_kernel(WindowArgs A) {
    const bool packed = A.cu_q != nullptr;
    int id = (int)blockIdx.x;
    const int key = id % A.mask.sinks; id /= A.mask.sinks;
    const int kv = id % A.kv_heads, b = id / A.kv_heads;
    Seq s;
    s.b = b;
    if (packed) {
        auto at = [&](const int32_t *cu, int i, int64_t lo, int64_t hi) { return min(max((int64_t)cu[i], lo), hi); };
        s.q0 = at(A.cu_q, b, 0, A.q_len);
        s.k0 = at(A.cu_k, b, 0, A.k_len);
        s.nq = (int)(at(A.cu_q, b + 1, s.q0, A.q_len) - s.q0);
        s.nk = (int)(at(A.cu_k, b + 1, s.k0, A.k_len) - s.k0);
    } else {
        s.q0 = s.k0 = 0;
        s.nq = (int)A.q_len;
        s.nk = (int)A.k_len;
    }
    if (key >= s.nk) return;
    const int end = window_end(A, s, min((key / A.block_keys + 1) * A.block_keys, s.nk) - 1);      // of the key's block
    for (int e = threadIdx.x; e < 2 * A.dim; e += 64) {
        const int64_t x = (int64_t)(e / A.dim * A.mask.sinks + key) * A.dim + e % A.dim;       // keys' gradients, then values'
        float sum = part_of(A, b, kv)[x];
        // the chunks that hold queries behind the window's last, in order, eight on their way at a time
        const int c0 = max(0, end + 1) / A.chunk, c1 = end + 1 < s.nq ? (s.nq - 1) / A.chunk : -1;
        for (int c = c0; c <= c1; c += 8) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = part_of(A, chunk_slot(A, s, packed, min(c + i, c1)), kv)[x];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i <= c1) sum += y[i];
        }
        const Rows &R = e < A.dim ? A.dk : A.dv;
        seq_base<T>(R, s, s.k0, packed, kv)[key * R.row + e % A.dim] = narrow<T>(e < A.dim ? sum * A.scale : sum);
    }
}

struct GradKernels {
    const void *delta, *q, *kv, *join;
    int keys, threads, q_rows, q_threads;    // of a block of kv and of q
};
template <typename T, int DP, int KG, int PG> static void use_kv(GradKernels &g, bool direct) {
    g.kv = direct ? (const void *)grad_kv_kernel<T, DP, KG, PG, true> : (const void *)grad_kv_kernel<T, DP, KG, PG, false>;
    g.keys = KvShape<T, DP, KG, PG>::KEYS;
    g.threads = KvShape<T, DP, KG, PG>::THREADS;
}
template <typename T, int DP, int MG, int PG, int SUB> static void use_q(GradKernels &g, bool direct) {
    g.q = direct ? (const void *)grad_q_kernel<T, DP, MG, PG, SUB, true> : (const void *)grad_q_kernel<T, DP, MG, PG, SUB, false>;
    g.q_rows = QShape<T, DP, MG, PG, SUB>::ROWS;
    g.q_threads = QShape<T, DP, MG, PG, SUB>::THREADS;
}
// few: there are not enough keys to keep the compute units busy with blocks of the large shape; blocks of 32 keys then, whose
// waves share out the queries.  few_q: the same of the queries.  Step of 512 tokens, 8 heads over 2 of 128 in bf16, with
// blocks of 32 keys 67 us, of 128 keys 95; of 8192 tokens 324 and 254.  32-bit tiles of 128 leave no room for a fourth wave,
// and the small shape is then never faster (2048 tokens: 1135 and 1071 us); of 64 it is (1024 tokens, 8 heads: 107 and 142).
template <typename T, int DP> static GradKernels grads_for(bool direct_q, bool direct_kv, bool few, bool few_q) {
    GradKernels g = {};
    g.delta = (const void *)delta_kernel<T>;
    g.join = (const void *)join_kernel<T>;
    constexpr int ALL = sizeof(T) == 2 || DP == 64 ? 4 : 2;          // waves whose tiles fit into LDS
    if constexpr (ALL == 4) {
        if (few) use_kv<T, DP, 1, 4>(g, direct_kv);
        else use_kv<T, DP, sizeof(T) == 2 ? 4 : 2, 2>(g, direct_kv);
    } else {
        use_kv<T, DP, 2, 2>(g, direct_kv);
    }
    if (few_q) use_q<T, DP, 1, ALL, 1>(g, direct_q);
    else use_q<T, DP, 4, 1, sizeof(T) == 2 ? 2 : 1>(g, direct_q);
    return g;
}
template <typename T> static GradKernels grads_of(int dim, bool direct_q, bool direct_kv, bool few, bool few_q) {
    return dim <= 64   ? grads_for<T, 64>(direct_q, direct_kv, few, few_q)
           : dim <= 96 ? grads_for<T, 96>(direct_q, direct_kv, few, few_q)
                       : grads_for<T, 128>(direct_q, direct_kv, few, few_q);
}

// Queries of a part: a step of 4096 tokens, 8 heads over 2 of 128 in bf16 under a window of 1024 takes 175 us with 512, 178 with
// 256 and 384, 208 with 1024, 421 without parts; in 32 bits 1084, 1091, 1082 and 3618.
constexpr int CHUNK = 512;
// Workspace: two floats a query row and head, then the first keys' parts where they are split.
struct GradWork { int64_t stats, part, total; int chunk; };
static int grad_work(const spmm_attn_desc_t *a, const char *where, bool packed, GradWork *w) {
    const int64_t n = packed ? 1 : a->batch;
    if (n && a->q_len > (INT64_C(1) << 44) / n / a->heads) return fail(SPMM_HIP_ERR_OVERFLOW, "%s: too many rows", where);
    w->stats = (n * a->q_len * a->heads * 8 + 15) / 16 * 16;
    w->chunk = 0;
    w->part = 0;
    const int64_t span = ((int64_t)a->window + 128 + 63) / 64 * 64;         // queries of an ordinary block of 128 keys
    // Where a sequence is longer than that, its first keys have queries beyond (2048 tokens under a window of 1024 with parts:
    // 152 us, without: 218; 257 tokens under one of 100 in 32 bits: 84 and 91); a mean of the lengths, as the offsets are not
    // known here, so a long sequence among many short ones is not split (4096 tokens alone: 421 us for 175), right but slower.
    const int64_t mean = packed && a->batch ? a->q_len / a->batch : a->q_len;
    if (a->window > 0 && a->window < a->k_len && a->sinks > 0 && a->sinks <= 128 && a->k_len > a->sinks && mean > span) {
        w->chunk = CHUNK;
        const int64_t slots = a->batch + (packed ? a->q_len / w->chunk + a->batch : a->batch * ((a->q_len + w->chunk - 1) / w->chunk));
        w->part = slots * a->kv_heads * 2 * a->sinks * a->dim * 4;
    }
    w->total = w->stats + w->part;
    return SPMM_HIP_OK;
}

}  // namespace attn

using namespace attn;

extern "C" int spmm_attn_window_work(const spmm_attn_desc_t *a, int32_t packed, size_t *bytes) {
    const int st = check_desc(a, "attn_window_work");
    if (st != SPMM_HIP_OK) return st;
    if (!bytes) return fail(SPMM_HIP_ERR_ARG, "attn_window_work: bytes is NULL");
    GradWork w;
    const int sw = grad_work(a, "attn_window_work", packed != 0, &w);
    if (sw == SPMM_HIP_OK) *bytes = (size_t)w.total;
    return sw;
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
    if (nb == 0 || (a->batch == 0 && !a->zero_rest)) return SPMM_HIP_OK;
    GradWork w;
    if ((st = grad_work(a, W, packed, &w))) return st;
    if (w.total > 0) {
        if (a->q_len > 0 && (!lse || (uintptr_t)lse % 4)) return fail(SPMM_HIP_ERR_ARG, "%s: lse is NULL or not aligned", W);
        if (!work || (uintptr_t)work % 16 || work_bytes < (size_t)w.total)
            return fail(SPMM_HIP_ERR_ARG, "%s: the workspace needs %lld bytes, 16-byte aligned", W, (long long)w.total);
    }
    A.lse = const_cast<float *>(lse);
    A.stats = (float *)work;
    A.part = (float *)((char *)work + w.stats);
    A.chunk = w.chunk;
    int qt = 0, kt = 0, ct = 0;
    const bool direct = A.k.direct && A.v.direct, direct_kv = direct && A.q.direct && A.dout.direct;
    const bool few = (nb * a->k_len + 127) / 128 * a->kv_heads < 128, few_q = (nb * a->q_len + 127) / 128 * a->heads < 256;
    const GradKernels G = a->dtype == SPMM_ATTN_F32 ? grads_of<float>(a->dim, direct, direct_kv, few, few_q)
                          : a->dtype == SPMM_ATTN_F16 ? grads_of<_Float16>(a->dim, direct, direct_kv, few, few_q)
                                                      : grads_of<__bf16>(a->dim, direct, direct_kv, few, few_q);
    if (a->q_len > 0 && (st = tile_count(a, W, packed, a->q_len, G.q_rows, &qt))) return st;
    A.block_keys = G.keys;
    if (a->k_len > 0 && (st = tile_count(a, W, packed, a->k_len, G.keys, &kt))) return st;
    if (w.chunk && (st = tile_count(a, W, packed, a->q_len, w.chunk, &ct))) return st;
    OnDevice on(a->device, W);
    if (on.status) return on.status;
    void *args[] = {&A};
    const int64_t rows = nb * a->q_len * a->heads;
    if ((st = launch(G.delta, W, (rows + 15) / 16, 256, args, stream))) return st;
    A.tiles = qt;
    if ((st = launch(G.q, W, (int64_t)qt * a->heads, G.q_threads, args, stream))) return st;
    A.tiles = kt;
    const int64_t extra = w.chunk ? (int64_t)ct * ((A.mask.sinks + G.keys - 1) / G.keys) : 0;
    if ((st = launch(G.kv, W, (kt + extra) * a->kv_heads, G.threads, args, stream))) return st;
    return w.chunk ? launch(G.join, W, a->batch * a->kv_heads * A.mask.sinks, 64, args, stream) : SPMM_HIP_OK;
}
