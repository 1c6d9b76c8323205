// attn_common.hpp -- what the attention kernels share: element types, matrix-core fragments, tiles in LDS, the visible
// range of the mask, and the host side's checks.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "../../include/spmm_attn.h"

namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int WAVE = 64;

// ------------------------------------------------------------------------------------------------ element types
// frag<T>: the 8 values a lane gives to one matrix instruction of depth 16 (32x32) or 32 (16x16).  For a 32x32
// product lane l holds row (or column) l % 32 and depth 8 * (l / 32) + 0..7; the result has column l % 32 and rows
// 8 * (r / 4) + 4 * (l / 32) + r % 4 in register r.  float has no instruction of that depth: eight of depth 2 take
// value j of every lane in turn, which is the same product summed in another order, so one kernel serves every type.
template <typename T> using frag = T __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x16 mma32(frag<__bf16> a, frag<__bf16> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(frag<_Float16> a, frag<_Float16> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(frag<float> a, frag<float> b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x4 mma16(frag<__bf16> a, frag<__bf16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(frag<_Float16> a, frag<_Float16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(frag<float> a, frag<float> b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// A value that every lane of a wave holds alike, in scalar registers.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
template <typename T> __device__ __forceinline__ T *uniform(T *p) {
    const uint64_t x = (uint64_t)p;
    return (T *)((uint64_t)(uint32_t)uniform((int)x) | (uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32);
}

// Round to nearest even; the only narrowing in these kernels apart from the stores of results.
template <typename T> __device__ __forceinline__ T narrow(float x) { return (T)x; }

// float16 has normal numbers down to 2^-14 only, and a thousand weights below that next to the largest may make up a result
// (a first key with a high score and a value near 0 is not rare), so weights are formed as a multiple of themselves that its range
// has room for: 2^UP<T>(top) if the largest is 2^top.  The power is taken out with the sum of the weights, at no cost.
template <typename T> __host__ __device__ constexpr float UP(int top) { return std::is_same<T, _Float16>::value ? 15.f - top : 0.f; }

// One bit per 16-bit half (or the top bit of a word) set where the exponent is all ones.
template <typename T> __device__ __forceinline__ uint32_t not_finite(uint32_t w);
template <> __device__ __forceinline__ uint32_t not_finite<__bf16>(uint32_t w) {
    return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}
template <> __device__ __forceinline__ uint32_t not_finite<_Float16>(uint32_t w) {
    return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}
template <> __device__ __forceinline__ uint32_t not_finite<float>(uint32_t w) {
    return ((w & 0x7f800000u) + 0x00800000u) & 0x80000000u;
}
__device__ __forceinline__ bool finite_f(float x) { return fabsf(x) < INFINITY; }

// ------------------------------------------------------------------------------------------------ tiles in LDS
// A tile is R rows of DP elements, DP = 64, 96 or 128 (the head's width rounded up, the rest zero), stored at a pitch of
// 64 or 128 elements with its 16-byte pieces exchanged within the row so that both ways of reading it spread over the
// banks: 8 elements of 16 different rows (row fragments), and 64 bytes of 4 adjacent rows (transposed fragments).
template <typename T, int DP> struct Tile {
    static constexpr int PITCH = DP <= 64 ? 64 : 128;
    static constexpr int EL = 16 / (int)sizeof(T);          // elements of a 16-byte piece

    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (sizeof(T) == 2)
            return PITCH == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
        else
            return PITCH == 128 ? (row & 15) << 1 : (row & 7) << 1;
    }
    static __device__ __forceinline__ int at(int row, int el) {      // element index of (row, el)
        return row * PITCH + (((el / EL) ^ swizzle(row)) * EL) + el % EL;
    }
    // elements [el, el + 8) of a row; el a multiple of 8
    static __device__ __forceinline__ frag<T> row_frag(const T *t, int row, int el) {
        if constexpr (sizeof(T) == 2) {
            return *reinterpret_cast<const frag<T> *>(t + at(row, el));
        } else {
            const f32x4 a = *reinterpret_cast<const f32x4 *>(t + at(row, el));
            const f32x4 b = *reinterpret_cast<const f32x4 *>(t + at(row, el + 4));
            return frag<T>{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        }
    }
    // The transposed fragment of the 32 elements at el0 against rows r0 .. r0 + 15: lane l holds element el0 + l % 32
    // of rows r0 + 4 h + 0..3 and r0 + 8 + 4 h + 0..3 (h = l / 32) -- the order in which a 32x32 product leaves its
    // rows, so a product's result is the other operand of the next one with no move between lanes.
    // The 16-bit form is the LDS transposing read: in each group of 16 lanes, lane 4 j + c addresses 4 elements of row
    // j, and lane i receives element i of the 4 rows.
    static __device__ __forceinline__ frag<T> col_frag(const T *t, int r0, int el0, int lane) {
        const int h = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            const int el = el0 + (lane & 16) + (lane & 3) * 4, row = r0 + 4 * h + ((lane >> 2) & 3);
            const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(t + at(row, el)));
            const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(t + at(row + 8, el)));
            typedef short i16x8 __attribute__((ext_vector_type(8)));
            const i16x8 w = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
            return __builtin_bit_cast(frag<T>, w);
        } else {
            frag<T> f;
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = t[at(r0 + 8 * (j >> 2) + 4 * h + (j & 3), el0 + (lane & 31))];
            return f;
        }
    }
};

// Buffer loads that write LDS: lane l fills the l-th 16 (or 4) bytes from `tile` on with those at byte `off` of the buffer,
// zeros where that lies outside.  The compiler does not count these loads: LDS is read after arrived<n>() (all of this
// wave's but the last n are there) and a barrier, and a wave has waited for all before it ends.  (With the builtin
// it does count them, and waits for every one of them before the next transposing read of any tile.)
// m0 says where in LDS; a load may read it one wait state after it is written, and scalar registers that a vector
// instruction wrote (readfirstlane) five after that.  The compiler does not look into the text, so the text waits, and names m0
// as written.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"          // that m0 is the compiler's own: it is named for the order with its uses
struct Buffer {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    i32x4 rsrc;
    __device__ __forceinline__ Buffer(const void *base, int bytes) {
        const uint64_t b = (uint64_t)base;
        rsrc = i32x4{uniform((int)b), uniform((int)(b >> 32)) & 0xffff, uniform(bytes), 0x00027000};
    }
    // where in LDS: the low half of the address
    static __device__ __forceinline__ int place(const void *tile) { return uniform((int)(uint32_t)(uintptr_t)tile); }
    __device__ __forceinline__ void to_lds16(void *tile, int off) const {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(place(tile)), "v"(off), "s"(rsrc) : "memory", "m0");
    }
    __device__ __forceinline__ void to_lds4(void *tile, int off) const {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(place(tile)), "v"(off), "s"(rsrc) : "memory", "m0");
    }
};
#pragma clang diagnostic pop
template <int LEFT = 0> __device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory"); }

// Brings the R rows of a tile from memory to LDS, THREADS threads together.
template <typename T, int DP, int R, int THREADS> struct Mover {
    using L = Tile<T, DP>;
    static constexpr int PP = L::PITCH / L::EL;             // 16-byte places of a row
    static constexpr int N = R * PP / THREADS, STEP = THREADS / PP;      // loads a thread, rows between them
    static_assert(R * PP % THREADS == 0 && THREADS % 64 == 0 && STEP > 0, "whole waves of pieces");
    static constexpr bool SAME = STEP % 16 == 0;            // the exchange within a row repeats every 16 rows
    int off[SAME ? 1 : N];                                  // byte offset of this thread's pieces from the tile's row 0

    // By buffer loads that write LDS: lane l of a wave fills place l of 64 consecutive ones, so the exchange of
    // pieces within a row is in which piece a lane asks for.  The buffer ends with the last row that is there, so what
    // lies behind it, and the pieces beyond dim, arrive as zeros without a comparison.  Rows are 16-byte aligned, dim
    // is a multiple of a piece and R rows span less than 2^31 bytes (Rows::direct).
    __device__ __forceinline__ void start(int tid, int dim, int64_t row) {
#pragma unroll
        for (int i = 0; i < (SAME ? 1 : N); ++i) {
            const int p = tid + i * THREADS, r = p / PP, e = ((p % PP) ^ L::swizzle(r)) * L::EL;
            off[i] = e < dim ? (r * (int)row + e) * (int)sizeof(T) : INT32_MIN;
        }
    }
    // rows: those left from `base` on (uniform).  The tile is there after arrived() and a barrier.
    __device__ __forceinline__ void send(int wave, T *tile, const T *base, int64_t row, int rows, int dim) const {
        const int n = min(rows, R);
        const Buffer buf(base, n > 0 ? ((n - 1) * (int)row + dim) * (int)sizeof(T) : 0);
#pragma unroll
        for (int i = 0; i < N; ++i)
            buf.to_lds16(tile + (i * THREADS + wave * 64) * L::EL, SAME ? off[0] + i * STEP * (int)row * (int)sizeof(T) : off[i]);
    }

    // Through registers, element by element: any alignment and width.
    template <typename F> static __device__ __forceinline__ void copy(int tid, int dim, T *tile, F row) {
#pragma unroll 1
        for (int p = tid; p < R * PP; p += THREADS) {
            const int r = p / PP, e = ((p % PP) ^ L::swizzle(r)) * L::EL;
            const T *src = row(r);
            T tmp[L::EL];
#pragma unroll
            for (int j = 0; j < L::EL; ++j) tmp[j] = src && e + j < dim ? src[e + j] : (T)0.f;
            uint4 w;
            __builtin_memcpy(&w, tmp, 16);
            *reinterpret_cast<uint4 *>(tile + p * L::EL) = w;
        }
    }
    // Of the pieces that this thread brought (arrived, or copied).
    static __device__ __forceinline__ bool any_not_finite(int tid, const T *tile) {
        uint32_t b = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint4 w = *reinterpret_cast<const uint4 *>(tile + (tid + i * THREADS) * L::EL);
            b |= not_finite<T>(w.x) | not_finite<T>(w.y) | not_finite<T>(w.z) | not_finite<T>(w.w);
        }
        return b != 0;
    }
};

// Fragments straight from memory (a wave's own 32 rows): elements [el, el + 8) of `src`, zero beyond dim or src null.
template <typename T> __device__ __forceinline__ frag<T> load_frag(const T *src, int el, int dim, bool wide) {
    frag<T> f = {};
    if (!src || el >= dim) return f;
    if (wide && el + 8 <= dim) {
        if constexpr (sizeof(T) == 2) {
            f = *reinterpret_cast<const frag<T> *>(src + el);
        } else {
            const f32x4 a = *reinterpret_cast<const f32x4 *>(src + el), b = *reinterpret_cast<const f32x4 *>(src + el + 4);
            f = frag<T>{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (el + j < dim) f[j] = src[el + j];
    }
    return f;
}

// The fragments are in their registers from here on.  Without it the compiler puts the wait for these loads where they are
// first used, in the loop, and there it waits on every turn for the tiles under way as well.
template <typename T, int N> __device__ __forceinline__ void settled(frag<T> (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// 4 consecutive results of a row
template <typename T> __device__ __forceinline__ void store4(T *dst, int el, int dim, bool wide, f32x4 x) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    if (el >= dim) return;
    const t4 v = {narrow<T>(x[0]), narrow<T>(x[1]), narrow<T>(x[2]), narrow<T>(x[3])};
    if (wide) {
        *reinterpret_cast<t4 *>(dst + el) = v;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (el + j < dim) dst[el + j] = v[j];
    }
}

// ------------------------------------------------------------------------------------------------ the mask
struct Mask {
    int window, sinks;      // window 0: none (sinks then has no effect)
    __device__ __forceinline__ bool sees(int p, int j) const {
        return j <= p && (window == 0 || p - j < window || j < sinks);
    }
    // every (p, j) of [p0, p1] x [j0, j1] visible
    __device__ __forceinline__ bool all(int p0, int p1, int j0, int j1) const {
        return j1 <= p0 && (window == 0 || p1 - j0 < window || j1 < sinks);
    }
};

// ------------------------------------------------------------------------------------------------ sequences
struct Seq {
    int64_t q0, k0;      // first row (packed) -- 0 without offsets
    int nq, nk, b;       // queries, keys, number of the sequence
    int tile;            // tile of the sequence; -1: behind the last tile (nq is then the number of tiles)
    int64_t rest;        // first row behind the last sequence (packed, tile == -1)
};

// Which tile of which sequence is tile number t, `rows` rows of the tiled side (queries or keys) a tile.  Without offsets
// by division; with offsets every wave sums the tiles of 64 sequences at a time.  Offsets are clamped into the
// buffers, so bad ones give wrong rows but no access outside.
__device__ __forceinline__ Seq find_tile_any(int t, int rows, bool by_key, const int32_t *cu_q, const int32_t *cu_k,
                                         int64_t batch, int64_t q_len, int64_t k_len) {
    Seq s;
    s.rest = 0;
    if (!cu_q) {
        const int64_t n = by_key ? k_len : q_len;
        const int per = (int)((n + rows - 1) / rows);
        s.b = per ? t / per : 0;
        s.tile = per && s.b < batch ? t % per : -1;
        s.q0 = s.k0 = 0;
        s.nq = (int)q_len;
        s.nk = (int)k_len;
        return s;
    }
    const int lane = threadIdx.x & (WAVE - 1);
    const int32_t *cu = by_key ? cu_k : cu_q;
    const int64_t lim = by_key ? k_len : q_len;
    int before = 0;
    int64_t last = 0;
    for (int64_t b0 = 0; b0 < batch; b0 += WAVE) {
        const int64_t b = b0 + lane;
        int64_t lo = 0, hi = 0;
        if (b < batch) {
            lo = min(max((int64_t)cu[b], (int64_t)0), lim);
            hi = min(max((int64_t)cu[b + 1], lo), lim);
        }
        const int mine = (int)((hi - lo + rows - 1) / rows);
        int incl = mine;
#pragma unroll
        for (int d = 1; d < WAVE; d *= 2) {
            const int o = __shfl_up(incl, d);
            if (lane >= d) incl += o;
        }
        const unsigned long long hit = __ballot(before + incl > t);
        if (hit) {
            const int src = __ffsll(hit) - 1;
            s.b = __builtin_amdgcn_readfirstlane((int)b0 + src);
            s.tile = __builtin_amdgcn_readfirstlane(t - before - __shfl(incl - mine, src));
            const int q0 = (int)min(max((int64_t)cu_q[s.b], (int64_t)0), q_len);
            const int k0 = (int)min(max((int64_t)cu_k[s.b], (int64_t)0), k_len);
            s.q0 = __builtin_amdgcn_readfirstlane(q0);
            s.k0 = __builtin_amdgcn_readfirstlane(k0);
            s.nq = __builtin_amdgcn_readfirstlane((int)min(max((int64_t)cu_q[s.b + 1], (int64_t)q0), q_len) - q0);
            s.nk = __builtin_amdgcn_readfirstlane((int)min(max((int64_t)cu_k[s.b + 1], (int64_t)k0), k_len) - k0);
            return s;
        }
        before += __shfl(incl, WAVE - 1);
        const int64_t top = __shfl(hi, (int)min((int64_t)WAVE, batch - b0) - 1);
        last = max(last, top);
    }
    s.tile = -1;
    s.b = 0;
    s.q0 = s.k0 = 0;
    s.nq = before;
    s.nk = 0;
    s.rest = last;
    return s;
}

// The same, in scalar registers: what depends on it are then branches and addresses of the whole wave.
__device__ __forceinline__ Seq find_tile(int t, int rows, bool by_key, const int32_t *cu_q, const int32_t *cu_k,
                                         int64_t batch, int64_t q_len, int64_t k_len) {
    Seq s = find_tile_any(t, rows, by_key, cu_q, cu_k, batch, q_len, k_len);
    s.q0 = uniform((int)s.q0);
    s.k0 = uniform((int)s.k0);
    s.nq = uniform(s.nq);
    s.nk = uniform(s.nk);
    s.b = uniform(s.b);
    s.tile = uniform(s.tile);
    s.rest = uniform((int)s.rest);
    return s;
}

// ------------------------------------------------------------------------------------------------ host side
struct Rows {             // spmm_attn_rows for a kernel
    char *ptr;
    int64_t seq, row, head;
    bool wide;            // 16-byte (inputs) or 4-element (outputs) accesses allowed
    bool direct;          // wide, rows apart by dim or more, and 128 rows span less than 2^31 bytes
};

extern thread_local char g_detail[256];
int fail(int status, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
int check_desc(const spmm_attn_desc_t *a, const char *where);
size_t elem_size(int dtype);
// An operand: a pointer if it has elements, not overlapping if written; out: kernel form with the alignment looked at.
int check_rows(const spmm_attn_desc_t *a, const spmm_attn_rows_t *r, const char *where, const char *name, int64_t batch,
               int64_t rows, int heads, bool written, Rows *out);
int launch(const void *kernel, const char *where, int64_t blocks, int threads, void **args, void *stream);

struct OnDevice {         // the call's device, and the caller's back
    int prev = -1, status = SPMM_HIP_OK;
    OnDevice(int device, const char *where);
    ~OnDevice();
};

}  // namespace attn
