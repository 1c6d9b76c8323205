// attn_paged.hip -- attention of one new token a sequence over keys and values in pages, and the write of new rows
// into the pages (include/spmm_attn.h).
//
// Each visible key and value is read once from memory and used by up to 16 query heads of its group, so bytes bound the
// kernel and it is laid out for loads that go straight into the matrix instructions, with no LDS on the way (larger groups
// read them again for every 16: 16 sequences of 16384 keys, 16 heads over 1 of 128 in bf16 37 us, 32 heads 54, 64 heads 90):
//  - a wave takes 16 keys at a time; S^T = K Q^T (16 keys x up to 16 heads) has a lane's 16-byte piece of one key's row
//    as its first operand;
//  - S^T leaves a lane with keys 4 (l / 16) + r, r = 0..3, of head l % 16.  exp(S^T) is then, as it stands, the first
//    operand of a 16x16x16 product (of four 16x16x4 ones in 32 bits), whose second operand is element j of value rows
//    4 (l / 16) + 0..3: lane l % 16 loads a piece of those four rows, and element j of each makes up product j.  The
//    values need no transposition.  16-bit products take the weights in two parts, so they lose nothing by rounding.
// A block's four waves share a stretch of the keys and join through LDS.  Where sequences are longer than a block should
// take alone, all of them are cut into parts of about one length by what the lengths say, as many as the compute units
// hold at once, and a second kernel joins the parts of a sequence in order.
// 32 sequences of 9843 to 16384 keys, 64 heads over 8 of 128 in bf16: 340 us, 5.05 TB/s (a large copy moves 4.7, a large
// sum reads 4.0).  A second set of registers for the next tile made that 340 from 325 in an earlier form, and nothing
// faster: with four blocks a compute unit there is enough on its way.
#include "attn_common.hpp"

namespace attn {

constexpr int PW = 4;                        // waves of a block
constexpr int PK = 16;                       // keys a wave takes at a time
constexpr int ALONE = 256;                   // keys up to which nothing is cut: a second launch costs more
constexpr int SPLIT_MIN = 64;                // keys a block takes at least otherwise: one tile a wave
constexpr int SPLIT_MAX = 256;               // parts of a sequence at most
// blocks that a compute unit holds at once
__host__ __device__ constexpr int paged_blocks(bool half) { return half ? 4 : 3; }

struct PagedArgs {
    Rows q, out;
    const char *k, *v;
    int64_t pages, page_rows, k_page, k_row, k_head, v_page, v_row, v_head, table_cols, table_stride;
    const int32_t *table, *lengths;
    bool k_wide, v_wide;
    int64_t batch, limit;                    // limit: longest sequence allowed
    int heads, kv_heads, dim, window, sinks, page_shift;      // page_shift: of a power of two, else -1
    int room, cap;                           // parts wanted of all sequences (0: they are not cut), and room for them
    float scale2;
    int32_t *start;                          // [batch][2] of a sequence: its first part, and how many
    float *lse, *part;                       // part: [heads][cap][2] max, sum, then [heads][cap][dim] weighted values
};

// The 16-key tiles that hold visible keys: `first` tiles from position 0, then those from `start` on.
struct Span {
    int first, start, tiles;
    __device__ __forceinline__ int at(int i) const { return (i < first ? i : start + i - first) * PK; }
};
__device__ __forceinline__ Span span_of(int len, int window, int sinks) {
    Span s;
    const int lo = window && len > window ? len - window : 0;
    s.start = lo / PK;
    s.first = min((min(sinks, len) + PK - 1) / PK, s.start);
    s.tiles = s.first + (len + PK - 1) / PK - s.start;
    return s;
}

// The cut of the sequences into parts: each into equal ones of `per` tiles at most, SPLIT_MAX of them at most.  Every wave
// works it out from the lengths.  With per = total / room + 1 there are room + batch parts at most.  With up to 64 sequences
// it is the smallest, but for 3 %, that makes them `room`, if 2 per does: a few blocks more than the compute units hold at
// once would take as long again, and a longer part is what the others wait for.  Next to as many parts for every
// sequence this costs about 2 us and gains where lengths differ: 17 sequences of 1 to 23493 keys, 32 heads over 4 of 96 in 32
// bits, 206 -> 68 us, 9 of 7 to 19511, 8 heads over 8 of 96 in fp16, 64 -> 46; 1000 keys of one sequence 9.8 -> 11.3.
__device__ __forceinline__ int tiles_of(const PagedArgs &A, int64_t b) {
    const int len = b < A.batch ? A.lengths[b] : 0;
    return len < 0 || len > A.limit ? 0 : span_of(len, A.window, A.sinks).tiles;
}
__device__ __forceinline__ int parts_of(int tiles, int per) {
    return min(max(1, (int)(((uint32_t)tiles + per - 1) / (uint32_t)per)), SPLIT_MAX);
}
// first: tiles of sequence `lane`
__device__ __forceinline__ int plan(const PagedArgs &A, int lane, int first) {
    if (A.batch <= WAVE) {
        // A sequence has 2^26 tiles and a few at most: the sum of 64 takes more than 32 bits, and with 2^27 a part none is cut.
        uint32_t low = first & 0xffff, high = (uint32_t)first >> 16;
#pragma unroll
        for (int d = 32; d; d /= 2) {
            low += __shfl_xor(low, d);
            high += __shfl_xor(high, d);
        }
        const uint64_t total = ((uint64_t)(uint32_t)uniform((int)high) << 16) + (uint32_t)uniform((int)low);
        const uint64_t each = total >> 32 ? total / (uint32_t)A.room : (uint32_t)total / (uint32_t)A.room;
        const int lo = max(SPLIT_MIN / PK, (int)min(each, (uint64_t)1 << 27) + 1);
        auto fits = [&](int per) {
            const int n = lane < A.batch ? parts_of(first, per) : 0;      // 256 at most
            int sum = 0;
#pragma unroll
            for (int bit = 0; bit <= 8; ++bit) sum += __popcll(__ballot(n >> bit & 1)) << bit;
            return sum <= A.room;
        };
        if (fits(lo) || !fits(2 * lo)) return lo;
        int per = 2 * lo;
        for (int step = lo / 2, i = 0; i < 5 && step > 0; step /= 2, ++i)
            if (fits(per - step)) per -= step;
        return per;
    }
    int64_t total = first;
    for (int64_t b = lane + WAVE; b < A.batch; b += WAVE) total += tiles_of(A, b);
#pragma unroll
    for (int d = 32; d; d /= 2) total += __shfl_xor(total, d);
    return uniform(max(SPLIT_MIN / PK, (int)min(total / A.room, (int64_t)INT32_MAX - 1) + 1));
}

// Depth 16: lane l gives row (column) l % 16 at depths 4 (l / 16) + 0..3.
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mma16x16(bf16x4 a, bf16x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4, a), __builtin_bit_cast(i16x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16x16(f16x4 a, f16x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
}

__device__ __align__(16) const float zero_row[SPMM_ATTN_MAX_DIM] = {};

// E elements of a row from element e on, zero beyond dim; `row` is zero_row where there is none.
template <typename T, int E> struct Piece {
    typedef T vec __attribute__((ext_vector_type(E)));
    static __device__ __forceinline__ vec load(const T *row, int e, int dim, bool wide) {
        if (wide) return *reinterpret_cast<const vec *>(e < dim ? row + e : (const T *)zero_row);
        vec v;
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = e + j < dim ? row[e + j] : (T)0.f;
        return v;
    }
};

// o[j] += weights (16 heads x 16 keys, as the scores' product leaves them) x column j of the lanes' pieces of the values.
template <typename T, int VE>
__device__ __forceinline__ void add_values(f32x4 (&o)[VE], const f32x4 &w, const typename Piece<T, VE>::vec (&v)[4]) {
    if constexpr (sizeof(T) == 2) {
        typedef T t4 __attribute__((ext_vector_type(4)));
        t4 hi, lo;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            hi[r] = narrow<T>(w[r]);
            lo[r] = narrow<T>(w[r] - (float)hi[r]);
        }
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const t4 b = {v[0][j], v[1][j], v[2][j], v[3][j]};
            o[j] = mma16x16(hi, b, o[j]);
            o[j] = mma16x16(lo, b, o[j]);
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < VE; ++j) o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[r], v[r][j], o[j], 0, 0, 0);
    }
}

// Values that are not finite, taken out of the pieces and summed by themselves in a wave's `extra`, a number a column: with a weight
// that was rounded to 0, or as its remainder is, and in a rescaling by 0, a product would make NaN of an infinity.
template <typename T, int VE> __device__ __forceinline__ void take_not_finite(float *extra, typename Piece<T, VE>::vec (&v)[4], int lane) {
#pragma unroll
    for (int j = 0; j < VE; ++j) {
        float x = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (!finite_f((float)v[r][j])) {
                x += (float)v[r][j];
                v[r][j] = (T)0.f;
            }
        x += __shfl_xor(x, 16);
        x += __shfl_xor(x, 32);
        if (lane < 16 && x != 0.f) extra[lane * VE + j] += x;
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(PW * 64, paged_blocks(sizeof(T) == 2)) void paged_kernel(PagedArgs A) {
    // a lane's columns of the values: VE from VE (lane % 16) on
    constexpr int NS = DP / 32, VE = DP / 16;
    constexpr float LIFT = UP<T>(0);                        // weights and their sums are 2^LIFT times as large
    const int group = A.heads / A.kv_heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, h4 = lane >> 4;
    const int hb = (group + 15) / 16;                       // blocks of 16 query heads of a group
    int id = (int)blockIdx.x;
    const int kv = id % A.kv_heads; id /= A.kv_heads;
    const int g0 = id % hb * 16; id /= hb;
    int64_t b = id;
    int per = 0, split = 0, parts = 1;                      // tiles of a part, which one this is, of how many
    if (A.room) {
        const int first = tiles_of(A, lane), part_tile = plan(A, lane, first);
        int before = 0;
        for (b = 0;; b += WAVE) {
            if (b >= A.batch) return;                       // fewer parts than there could be
            const int tiles = b ? tiles_of(A, b + lane) : first, n0 = b + lane < A.batch ? parts_of(tiles, part_tile) : 0;
            int incl = n0;
#pragma unroll
            for (int d = 1; d < WAVE; d *= 2) {
                const int o = __shfl_up(incl, d);
                if (lane >= d) incl += o;
            }
            const unsigned long long hit = __ballot(before + incl > id);
            if (hit) {
                const int src = __ffsll(hit) - 1;
                b += src;
                split = uniform(id - before - __shfl(incl - n0, src));
                parts = uniform(__shfl(n0, src));
                per = (uniform(__shfl(tiles, src)) + parts - 1) / parts;
                if (split == 0 && kv == 0 && g0 == 0 && threadIdx.x == 0) {
                    A.start[2 * b] = id;
                    A.start[2 * b + 1] = parts;
                }
                break;
            }
            before += uniform(__shfl(incl, WAVE - 1));
        }
    }

    int len = A.lengths[b];
    bool bad = len < 0 || len > A.limit;
    if (bad) len = 0;
    const Span sp = span_of(len, A.window, A.sinks);
    const int t0 = split * per, t1 = A.room ? min(t0 + per, sp.tiles) : sp.tiles;

    const int head = kv * group + g0 + n;
    const bool mine = g0 + n < group;
    frag<T> qf[NS];
    {
        const T *qr = mine ? (const T *)A.q.ptr + b * A.q.seq + head * A.q.head : nullptr;
#pragma unroll
        for (int s = 0; s < NS; ++s) qf[s] = load_frag<T>(qr, s * 32 + h4 * 8, A.dim, A.q.wide);
    }
    const T *kb = (const T *)A.k + kv * A.k_head, *vb = (const T *)A.v + kv * A.v_head;
    const int32_t *table = A.table + b * A.table_stride;
    auto seen = [&](int j) { return j < len && (A.window == 0 || len - 1 - j < A.window || j < A.sinks); };
    // page and row of this lane's key n of tile t; the page is -1 if the key is not seen
    auto locate = [&](int t, int &slot) -> int {
        const int j = t < t1 ? sp.at(t) + n : len;
        uint32_t c;
        if (A.page_shift >= 0) {
            c = (uint32_t)j >> A.page_shift;
            slot = j - (int)(c << A.page_shift);
        } else {
            c = (uint32_t)j / (uint32_t)A.page_rows;
            slot = j - (int)(c * (uint32_t)A.page_rows);
        }
        if (!seen(j)) return -1;
        const int pg = table[c];
        return pg < 0 || pg >= A.pages ? -2 : pg;
    };

    __shared__ float extra[PW][DP];
#pragma unroll
    for (int i = 0; i < DP; i += WAVE) extra[wave][i + lane] = 0.f;
    f32x4 o[VE];
    float m, sum;
    // A second time, and with care, if some sum is not finite in the end: each wave for itself.
    for (bool careful = false;; careful = true) {
#pragma unroll
        for (int j = 0; j < VE; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        m = -INFINITY;
        sum = 0.f;
        int slot_next, page_next = locate(t0 + wave, slot_next);
        for (int t = t0 + wave; t < t1; t += PW) {
            const int j0 = sp.at(t), page = page_next, slot = slot_next;
            page_next = locate(t + PW, slot_next);
            bad |= page == -2;
            const int64_t voff = page < 0 ? -1 : (int64_t)page * A.v_page + slot * A.v_row;
            const T *kr = page < 0 ? (const T *)zero_row : kb + (int64_t)page * A.k_page + slot * A.k_row;
            frag<T> kf[NS];
#pragma unroll
            for (int s = 0; s < NS; ++s) kf[s] = Piece<T, 8>::load(kr, s * 32 + h4 * 8, A.dim, A.k_wide);
            typename Piece<T, VE>::vec vr[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t off = __shfl(voff, 4 * h4 + r);
                vr[r] = Piece<T, VE>::load(off < 0 ? (const T *)zero_row : vb + off, n * VE, A.dim, A.v_wide);
            }
            f32x4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < NS; ++s) sc = mma16(kf[s], qf[s], sc);
            float mx = m;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                sc[r] = seen(j0 + 4 * h4 + r) ? sc[r] * A.scale2 : -INFINITY;
                mx = fmaxf(mx, sc[r]);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float base = mx == -INFINITY ? 0.f : mx;
            if (__any(mx != m)) {
                const float alpha = __builtin_amdgcn_exp2f(m - base);
                sum *= alpha;
                f32x4 a4;                                       // accumulator rows are heads 4 h4 + r
#pragma unroll
                for (int r = 0; r < 4; ++r) a4[r] = __shfl(alpha, 4 * h4 + r);
#pragma unroll
                for (int j = 0; j < VE; ++j) o[j] *= a4;
                m = mx;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                sc[r] = __builtin_amdgcn_exp2f(sc[r] - (base - LIFT));
                sum += sc[r];
            }
            if (careful) take_not_finite<T, VE>(extra[wave], vr, lane);
            add_values<T, VE>(o, sc, vr);
        }
        bool odd = false;
#pragma unroll
        for (int j = 0; j < VE; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) odd |= !finite_f(o[j][r]);
        if (careful || !__any(odd)) break;
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (__any(bad)) sum = __builtin_nanf("");

    // join the waves: in wave order
    __shared__ float sm[PW][16], ss[PW][16];
    __shared__ float so[PW][16][DP + 4];
    if (h4 == 0) {
        sm[wave][n] = m;
        ss[wave][n] = sum;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < VE; ++j) so[wave][4 * h4 + r][n * VE + j] = o[j][r];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * DP; i += PW * 64) {
        const int hh = i / DP, d = i % DP;
        if (g0 + hh >= group || d >= A.dim) continue;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < PW; ++w) mx = fmaxf(mx, sm[w][hh]);
        const float base = mx == -INFINITY ? 0.f : mx;
        float tot = 0.f, acc = 0.f, x = 0.f;                // x: 0, or not finite
#pragma unroll
        for (int w = 0; w < PW; ++w) x += extra[w][d];
#pragma unroll
        for (int w = 0; w < PW; ++w) {
            const float f = __builtin_amdgcn_exp2f(sm[w][hh] - base);
            tot += f * ss[w][hh];
            acc += f * so[w][hh][d];
        }
        const int hd = kv * group + g0 + hh;
        if (parts == 1) {
            ((T *)A.out.ptr)[b * A.out.seq + hd * A.out.head + d] = narrow<T>((tot == 0.f ? 0.f : acc / tot) + x);
            if (d == 0) A.lse[b * A.heads + hd] = tot == 0.f ? -INFINITY : (mx - LIFT) * LN2 + __logf(tot);
        } else {
            const int64_t at = (int64_t)hd * A.cap + id;
            if (d == 0) {
                A.part[2 * at] = mx;
                A.part[2 * at + 1] = tot;
            }
            A.part[2 * (int64_t)A.heads * A.cap + at * A.dim + d] = acc + x;
        }
    }
}

// A block a (sequence, head): its parts joined in an order that is fixed by their number.  Each of the four waves takes a
// quarter of them, eight parts on their way at a time.  What is not finite in a part is added to the result as it is.
constexpr int JW = 4;
template <typename T> __global__ __launch_bounds__(JW * 64) void paged_join_kernel(PagedArgs A) {
    const int64_t x = blockIdx.x, b = x / A.heads;
    const int hd = (int)(x % A.heads), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int splits = A.start[2 * b + 1];
    if (splits == 1) return;                                // the block that took it has stored the result
    const int64_t at = (int64_t)hd * A.cap + A.start[2 * b];
    const float *st = A.part + 2 * at, *p = A.part + 2 * (int64_t)A.heads * A.cap + at * A.dim;
    float mx = -INFINITY;
    for (int s = lane; s < splits; s += WAVE) mx = fmaxf(mx, st[2 * s]);
#pragma unroll
    for (int d = 32; d; d /= 2) mx = fmaxf(mx, __shfl_xor(mx, d));
    const float base = mx == -INFINITY ? 0.f : mx;
    float tot = 0.f, a0 = 0.f, a1 = 0.f, x0 = 0.f, x1 = 0.f;
    const int e0 = min(lane, A.dim - 1), e1 = min(lane + WAVE, A.dim - 1);
    const int per = (splits + JW - 1) / JW, last = min((wave + 1) * per, splits);
    for (int s0 = wave * per; s0 < last; s0 += WAVE) {
        const int n = min(WAVE, last - s0);
        const float *ps = p + (int64_t)s0 * A.dim;
        float f = 0.f, add = 0.f;
        if (lane < n) {
            f = __builtin_amdgcn_exp2f(st[2 * (s0 + lane)] - base);
            add = f * st[2 * (s0 + lane) + 1];
        }
#pragma unroll
        for (int d = 32; d; d /= 2) add += __shfl_xor(add, d);
        tot += add;
        for (int s = 0; s < n; s += 8) {
            float y0[8], y1[8];                             // all asked for before any is used; past the last part that one again
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float *pi = ps + min(s + i, n - 1) * A.dim;
                y0[i] = pi[e0];
                y1[i] = pi[e1];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(y0[i]), "+v"(y1[i]));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float fs = __shfl(f, s + i);
                const float g0 = finite_f(y0[i]) ? y0[i] : 0.f, g1 = finite_f(y1[i]) ? y1[i] : 0.f;
                a0 += fs * g0;                              // fs is 0 past the last part
                a1 += fs * g1;
                x0 += y0[i] - g0;
                x1 += y1[i] - g1;
            }
        }
    }
    __shared__ float wt[JW], w0[JW][WAVE], w1[JW][WAVE], wx0[JW][WAVE], wx1[JW][WAVE];
    if (lane == 0) wt[wave] = tot;
    w0[wave][lane] = a0;
    w1[wave][lane] = a1;
    wx0[wave][lane] = x0;
    wx1[wave][lane] = x1;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 1; i < JW; ++i) {
        tot += wt[i];
        a0 += w0[i][lane];
        a1 += w1[i][lane];
        x0 += wx0[i][lane];
        x1 += wx1[i][lane];
    }
    const float inv = tot == 0.f ? 0.f : 1.f / tot;
    T *dst = (T *)A.out.ptr + b * A.out.seq + hd * A.out.head;
    if (lane < A.dim) dst[lane] = narrow<T>(a0 * inv + x0);
    if (lane + WAVE < A.dim) dst[lane + WAVE] = narrow<T>(a1 * inv + x1);
    if (lane == 0) A.lse[x] = tot == 0.f ? -INFINITY : (mx - UP<T>(0)) * LN2 + __logf(tot);
}

// ------------------------------------------------------------------------------------------------ append
struct AppendArgs {
    Rows k, v;
    char *kp, *vp;
    const int32_t *cu;
    int64_t pages, page_rows, k_page, k_row, k_head, v_page, v_row, v_head, table_cols, table_stride;
    const int32_t *table, *lengths;
    int64_t batch, rows, es;
    int kv_heads, dim;
    bool k_wide, v_wide;
};

// 16 lanes a (row, head): it is moved whole, by 16-byte pieces where everything is aligned to them.  Bytes bound it: prompts of
// 30450 rows, 8 heads of 128 in bf16, 57 us, 4.4 TB/s read and written (a large copy: 4.7).
__global__ __launch_bounds__(256) void append_kernel(AppendArgs A) {
    const int64_t x = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (x >= A.rows * A.kv_heads) return;
    const int64_t row = x / A.kv_heads;
    const int head = (int)(x % A.kv_heads), l = threadIdx.x & 15;
    int64_t b = row, pos;
    if (A.cu) {
        int64_t lo = 0, hi = A.batch;                        // last sequence that starts at or before the row
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) / 2;
            if (A.cu[mid] <= row) lo = mid; else hi = mid;
        }
        b = lo;
        if (row < A.cu[b] || row >= A.cu[b + 1]) return;     // behind the last sequence
        pos = (int64_t)A.lengths[b] - A.cu[b + 1] + row;
    } else {
        pos = (int64_t)A.lengths[b] - 1;
    }
    if (pos < 0 || (A.lengths[b] - 1) / A.page_rows >= A.table_cols) return;
    const int64_t pg = A.table[b * A.table_stride + pos / A.page_rows];
    if (pg < 0 || pg >= A.pages) return;
    const int64_t slot = pos % A.page_rows;
    const char *ks = A.k.ptr + (row * A.k.row + head * A.k.head) * A.es, *vs = A.v.ptr + (row * A.v.row + head * A.v.head) * A.es;
    char *kd = A.kp + (pg * A.k_page + slot * A.k_row + head * A.k_head) * A.es;
    char *vd = A.vp + (pg * A.v_page + slot * A.v_row + head * A.v_head) * A.es;
    const int bytes = A.dim * (int)A.es;
    auto move = [&](char *d, const char *s, bool wide) {
        if (wide)
            for (int i = l * 16; i < bytes; i += 256) *(uint4 *)(d + i) = *(const uint4 *)(s + i);
        else
            for (int i = l * 2; i < bytes; i += 32) *(uint16_t *)(d + i) = *(const uint16_t *)(s + i);
    };
    move(kd, ks, A.k_wide);
    move(vd, vs, A.v_wide);
}

// ------------------------------------------------------------------------------------------------ host
static int check_pages(const spmm_attn_desc_t *a, const spmm_attn_pages_t *p, const char *where, bool written, bool *k_wide,
                       bool *v_wide) {
    if (!p) return fail(SPMM_HIP_ERR_ARG, "%s: no pages", where);
    if (p->pages < 0 || p->page_rows < 1 || p->table_cols < 0 || p->table_stride < 0)
        return fail(SPMM_HIP_ERR_ARG, "%s: %lld pages of %lld rows, %lld table columns", where, (long long)p->pages,
                    (long long)p->page_rows, (long long)p->table_cols);
    if (p->pages > INT32_MAX || p->page_rows > INT32_MAX / 2 || p->table_cols > (INT64_C(1) << 40))
        return fail(SPMM_HIP_ERR_OVERFLOW, "%s: sizes of the pages", where);
    if (a->batch > 1 && p->table_stride < p->table_cols && p->table_stride != 0)
        return fail(SPMM_HIP_ERR_ARG, "%s: the table's rows overlap", where);
    if (a->batch > 0 && (!p->lengths || (p->table_cols > 0 && !p->table) || (p->pages > 0 && (!p->k || !p->v))))
        return fail(SPMM_HIP_ERR_ARG, "%s: pages, table or lengths are NULL", where);
    if (((uintptr_t)p->table | (uintptr_t)p->lengths) % 4) return fail(SPMM_HIP_ERR_ARG, "%s: table or lengths are not aligned", where);
    // the same rules as for rows: (page, row, head) stand for (sequence, row, head)
    const spmm_attn_rows_t k = {p->k, p->k_page, p->k_row, p->k_head}, v = {p->v, p->v_page, p->v_row, p->v_head};
    Rows r;
    int st = check_rows(a, &k, where, "the key pages", p->pages, p->page_rows, a->kv_heads, written, &r);
    if (st == SPMM_HIP_OK) st = check_rows(a, &v, where, "the value pages", p->pages, p->page_rows, a->kv_heads, written, &r);
    if (st != SPMM_HIP_OK) return st;
    const int64_t el = 16 / (int64_t)elem_size(a->dtype);
    auto wide = [&](const void *ptr, int64_t s0, int64_t s1, int64_t s2) {
        return (uintptr_t)ptr % 16 == 0 && s0 % el == 0 && s1 % el == 0 && s2 % el == 0 && a->dim % el == 0;
    };
    *k_wide = wide(p->k, p->k_page, p->k_row, p->k_head);
    *v_wide = wide(p->v, p->v_page, p->v_row, p->v_head);
    return SPMM_HIP_OK;
}

// Parts wanted of all sequences (0: they are not cut) and the most there can be: as many blocks as are on the compute units at
// once (four each, three with 32-bit elements), each part of SPLIT_MIN keys or more, SPLIT_MAX a sequence at most.
// In bf16, 8 heads over 1 of 128: 1000 keys 11.3 us with parts of 64 keys, 1.4 more with 128, 4.4 with 256, 10 with 512; 2 key
// heads, 100000 keys 33 us with 256 parts, 4.5 more with 128 or 512.  Batch of 32 of 4096 keys, 32 heads over 8: 1024 blocks
// 111 us, 512 blocks 4 % more, 2048 blocks 3 %; in 32 bits 768 blocks 210, 512 blocks 250, 1024 280.
static void cut(const spmm_attn_desc_t *a, int64_t max_length, int *room, int64_t *parts) {
    const int64_t group = a->heads / a->kv_heads, each = a->kv_heads * ((group + 15) / 16);
    int64_t keys = max_length;
    if (a->window && a->window < keys) keys = (int64_t)a->window + (a->sinks < keys - a->window ? a->sinks : keys - a->window);
    *room = 0;
    *parts = a->batch;
    if (keys <= ALONE) return;
    const int64_t want = 256 * paged_blocks(a->dtype != SPMM_ATTN_F32) / each;
    *room = want > 1 ? (int)want : 1;
    // first keys and window: up to three tiles more than their number asks for
    const int64_t most = (keys + 3 * PK + SPLIT_MIN - 1) / SPLIT_MIN, n = a->batch * (most < SPLIT_MAX ? most : SPLIT_MAX);
    *parts = n < *room + a->batch ? n : *room + a->batch;
}

template <typename T> static const void *paged_of(int dim) {
    return dim <= 64 ? (const void *)paged_kernel<T, 64> : (const void *)paged_kernel<T, 128>;
}

}  // namespace attn

using namespace attn;

extern "C" int spmm_attn_paged_work(const spmm_attn_desc_t *a, int64_t max_length, size_t *bytes) {
    const int st = check_desc(a, "attn_paged_work");
    if (st != SPMM_HIP_OK) return st;
    if (!bytes || max_length < 0 || max_length > INT32_MAX / 2)
        return fail(SPMM_HIP_ERR_ARG, "attn_paged_work: bytes is NULL, or max_length %lld", (long long)max_length);
    int room;
    int64_t parts;
    cut(a, max_length, &room, &parts);
    *bytes = room ? (size_t)((a->batch + 1) / 2 * 4 + parts * a->heads * (a->dim + 2)) * 4 : 0;
    return SPMM_HIP_OK;
}

extern "C" int spmm_attn_paged(const spmm_attn_desc_t *a, const spmm_attn_rows_t *q, const spmm_attn_pages_t *pages,
                               int64_t max_length, const spmm_attn_rows_t *out, float *lse, void *work, size_t work_bytes,
                               void *stream) {
    const char *W = "attn_paged";
    PagedArgs A = {};
    int st = check_desc(a, W);
    if (st != SPMM_HIP_OK) return st;
    if ((st = check_rows(a, q, W, "q", a->batch, 1, a->heads, false, &A.q)) ||
        (st = check_rows(a, out, W, "out", a->batch, 1, a->heads, true, &A.out)) ||
        (st = check_pages(a, pages, W, false, &A.k_wide, &A.v_wide)))
        return st;
    size_t need = 0;
    if ((st = spmm_attn_paged_work(a, max_length, &need))) return st;
    if (a->batch == 0) return SPMM_HIP_OK;
    if (!lse || (uintptr_t)lse % 4) return fail(SPMM_HIP_ERR_ARG, "%s: lse is NULL or not aligned", W);
    if (need > 0 && (!work || (uintptr_t)work % 16 || work_bytes < need))
        return fail(SPMM_HIP_ERR_ARG, "%s: the workspace needs %zu bytes, 16-byte aligned", W, need);
    // keys are read in pieces of 8 elements, values in pieces of 4 or 8: none may pass the row's end
    A.k_wide = A.k_wide && a->dim % 8 == 0;
    A.v_wide = A.v_wide && a->dim % (a->dim <= 64 ? 4 : 8) == 0;
    A.k = (const char *)pages->k;
    A.v = (const char *)pages->v;
    A.pages = pages->pages;
    A.page_rows = pages->page_rows;
    A.k_page = pages->k_page;
    A.k_row = pages->k_row;
    A.k_head = pages->k_head;
    A.v_page = pages->v_page;
    A.v_row = pages->v_row;
    A.v_head = pages->v_head;
    A.table = pages->table;
    A.lengths = pages->lengths;
    A.table_cols = pages->table_cols;
    A.table_stride = pages->table_stride;
    A.batch = a->batch;
    A.limit = pages->table_cols > max_length / pages->page_rows ? max_length : pages->table_cols * pages->page_rows;
    A.heads = a->heads;
    A.kv_heads = a->kv_heads;
    A.dim = a->dim;
    A.window = a->window;
    A.sinks = a->window ? a->sinks : 0;
    int64_t parts;
    cut(a, max_length, &A.room, &parts);
    if (parts > INT32_MAX) return fail(SPMM_HIP_ERR_OVERFLOW, "%s: too many parts", W);
    A.cap = (int)parts;
    A.page_shift = A.page_rows & (A.page_rows - 1) ? -1 : __builtin_ctzll((unsigned long long)A.page_rows);
    A.scale2 = a->scale * LOG2E;
    A.lse = lse;
    A.start = (int32_t *)work;
    A.part = (float *)work + (a->batch + 1) / 2 * 4;
    OnDevice on(a->device, W);
    if (on.status) return on.status;
    const void *kern = a->dtype == SPMM_ATTN_F32 ? paged_of<float>(a->dim)
                       : a->dtype == SPMM_ATTN_F16 ? paged_of<_Float16>(a->dim) : paged_of<__bf16>(a->dim);
    const void *join = a->dtype == SPMM_ATTN_F32 ? (const void *)paged_join_kernel<float>
                       : a->dtype == SPMM_ATTN_F16 ? (const void *)paged_join_kernel<_Float16>
                                                   : (const void *)paged_join_kernel<__bf16>;
    void *args[] = {&A};
    const int64_t hb = (a->heads / a->kv_heads + 15) / 16;
    if ((st = launch(kern, W, parts * hb * a->kv_heads, PW * 64, args, stream))) return st;
    return A.room ? launch(join, W, a->batch * a->heads, JW * 64, args, stream) : SPMM_HIP_OK;
}

extern "C" int spmm_attn_append(const spmm_attn_desc_t *a, const spmm_attn_rows_t *k, const spmm_attn_rows_t *v,
                                const int32_t *cu, const spmm_attn_pages_t *pages, void *stream) {
    const char *W = "attn_append";
    AppendArgs A = {};
    int st = check_desc(a, W);
    if (st != SPMM_HIP_OK) return st;
    if ((uintptr_t)cu % 4) return fail(SPMM_HIP_ERR_ARG, "%s: offsets are not aligned", W);
    const int64_t rows = cu ? a->q_len : a->batch;
    bool kw, vw;
    if ((st = check_rows(a, k, W, "k", 1, rows, a->kv_heads, false, &A.k)) ||
        (st = check_rows(a, v, W, "v", 1, rows, a->kv_heads, false, &A.v)) ||
        (st = check_pages(a, pages, W, true, &kw, &vw)))
        return st;
    if (rows == 0 || a->batch == 0 || pages->pages == 0) return SPMM_HIP_OK;
    A.k_wide = A.k.wide && kw;
    A.v_wide = A.v.wide && vw;
    A.kp = (char *)pages->k;
    A.vp = (char *)pages->v;
    A.cu = cu;
    A.pages = pages->pages;
    A.page_rows = pages->page_rows;
    A.k_page = pages->k_page;
    A.k_row = pages->k_row;
    A.k_head = pages->k_head;
    A.v_page = pages->v_page;
    A.v_row = pages->v_row;
    A.v_head = pages->v_head;
    A.table = pages->table;
    A.lengths = pages->lengths;
    A.table_cols = pages->table_cols;
    A.table_stride = pages->table_stride;
    A.batch = a->batch;
    A.rows = rows;
    A.es = (int64_t)elem_size(a->dtype);
    A.kv_heads = a->kv_heads;
    A.dim = a->dim;
    OnDevice on(a->device, W);
    if (on.status) return on.status;
    void *args[] = {&A};
    return launch((const void *)append_kernel, W, (rows * a->kv_heads + 15) / 16, 256, args, stream);
}
