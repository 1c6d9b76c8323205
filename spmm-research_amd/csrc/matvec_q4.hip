// matvec_q4.hip -- products of a few vectors with 4-bit weights (include/spmm_q4.h).
//
// The weights are read once, half a byte each, and that is the kernel's time; everything else is kept under it.  A wave
// takes tiles of 16 rows x 128 columns, laid out as its lanes read them: one 16-byte load a lane is the first operand of
// four 16x16x32 products, whose second operand holds up to 16 vectors.  A nibble becomes 16 + q in the 16-bit type by
// two integer operations for two weights (its bits are put into the mantissa of 16.0, which is exact); a fifth operand of
// ones sums x over the same columns, so that with C = sum (16 + q) x and X = sum x a group adds
//     scale * (C - (16 + zero) X).
// 16 is the smallest such offset, so little is lost in that difference (2^-24 * 31 / |q - zero| relative to a group's
// sum of |w x|).  32-bit x is split into three bfloat16 parts of 8 bits each that sum to it exactly and take three of
// the 16 columns.
// Four vectors in fp16 with 16384 x 8192 weights in groups of 128 with zero points: 17.7 us, 4.0 TB/s; one in 32 bits with
// 512 x 512 in groups of 32: 6.6 us, nearly all of it the launch and two memory latencies.
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/spmm_q4.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
template <typename T> using frag = T __attribute__((ext_vector_type(8)));

constexpr int TR = 16, TC = 128;             // rows and columns of a tile, 1024 bytes
constexpr int WMAX = 16;                     // waves of a block

__device__ __forceinline__ f32x4 mma(frag<__bf16> a, frag<__bf16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(frag<_Float16> a, frag<_Float16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Type that enters the matrix unit, columns of it that one vector takes, and 16 + nibble: element 2 p of the 8 is nibble p
// of the word, element 2 p + 1 nibble p + 4, moved to the top mantissa bits of 16.0.
template <typename T> struct Kind;
template <> struct Kind<__bf16> {
    using M = __bf16;
    static constexpr int PARTS = 1, BIT = 3;
    static constexpr uint32_t BASE = 0x41804180u, MASK = 0x00780078u;
};
template <> struct Kind<float> : Kind<__bf16> { static constexpr int PARTS = 3; };
template <> struct Kind<_Float16> {
    using M = _Float16;
    static constexpr int PARTS = 1, BIT = 6;
    static constexpr uint32_t BASE = 0x4c004c00u, MASK = 0x03c003c0u;
};
template <typename T> __device__ __forceinline__ frag<typename Kind<T>::M> unpack(uint32_t w) {
    using K = Kind<T>;
    uint32_t u[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int sh = K::BIT - 4 * p;
        u[p] = ((sh >= 0 ? w << (sh & 31) : w >> (-sh & 31)) & K::MASK) | K::BASE;
    }
    const uint4 v = make_uint4(u[0], u[1], u[2], u[3]);
    return __builtin_bit_cast(frag<typename K::M>, v);
}

struct Args {
    const uint4 *w;                          // [row tiles][column tiles][64 lanes]
    const void *scales;                      // [row tiles][groups][16]
    const uint32_t *zeros;                   // [row tiles][groups][16] bytes, or null
    const char *x;
    char *y;
    int64_t rows, cols, x_stride, y_stride, tokens;
    int tiles, groups, row_tiles, group;     // column tiles; groups; row tiles; columns of a group
    bool wide;
};

// x[tok][k .. k + 7] as it stands in memory, zeros where there is none
template <typename T> __device__ __forceinline__ frag<T> fetch_x(const Args &A, int64_t tok, int64_t k, bool mine) {
    frag<T> f = {};
    if (!mine || k >= A.cols) return f;
    const T *p = (const T *)A.x + tok * A.x_stride + k;
    if (A.wide && k + 8 <= A.cols) {
        __builtin_memcpy(&f, __builtin_assume_aligned(p, 16), sizeof f);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (k + j < A.cols) f[j] = p[j];
    }
    return f;
}
// Part `part` of it as an operand
template <typename T> __device__ __forceinline__ frag<typename Kind<T>::M> part_x(const frag<T> &x, int part) {
    if constexpr (sizeof(T) == 2) {
        return x;
    } else {
        frag<__bf16> f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // 8 bits of the value at a time, cut off, so each rest is exact; an infinity or NaN is all in the first part
            float r = x[j];
            uint32_t hi = __builtin_bit_cast(uint32_t, r) & 0xffff0000u;
#pragma unroll
            for (int i = 1; i <= 2; ++i) {
                const float rest = (hi & 0x7f800000u) == 0x7f800000u ? 0.f : r - __builtin_bit_cast(float, hi);
                if (part >= i) {
                    r = rest;
                    hi = __builtin_bit_cast(uint32_t, r) & 0xffff0000u;
                }
            }
            if (part == 0 && r != r) hi |= 0x00400000u;
            f[j] = __builtin_bit_cast(__bf16, (uint16_t)(hi >> 16));
        }
        return f;
    }
}

// A block takes RT row tiles, its waves share out the column tiles; SG scales a column tile.
template <typename T, bool ZEROS, int RT, int SG> __global__ __launch_bounds__(WMAX * 64) void matvec_kernel(Args A) {
    using K = Kind<T>;
    using M = typename K::M;
    constexpr int PARTS = K::PARTS, PER = 16 / PARTS;        // vectors a block takes
    typedef T t4 __attribute__((ext_vector_type(4)));
    __shared__ float part[WMAX][TR][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, n = lane & 15, g4 = lane >> 4;
    const int rt0 = blockIdx.x * RT;
    const int64_t t0 = (int64_t)blockIdx.y * PER, tok = t0 + n / PARTS;
    const bool mine = n < PER * PARTS && tok < A.tokens;
    frag<M> one;
#pragma unroll
    for (int j = 0; j < 8; ++j) one[j] = (M)1.f;

    f32x4 y[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    // past the last row tile the last one again
    auto weights = [&](int t, uint4 (&w)[RT]) {
#pragma unroll
        for (int i = 0; i < RT; ++i) w[i] = A.w[((int64_t)min(rt0 + i, A.row_tiles - 1) * A.tiles + t) * 64 + lane];
    };
    uint4 ahead[RT];
    if (wave < A.tiles) weights(wave, ahead);
    for (int t = wave; t < A.tiles; t += waves) {
        // everything of the tile, and the next one's weights, is asked for before anything is used
        uint4 w[RT];
        t4 sc[RT][SG];
        uint32_t z[RT][SG];
        frag<T> xr[4];
#pragma unroll
        for (int i = 0; i < RT; ++i) w[i] = ahead[i];
#pragma unroll
        for (int s = 0; s < 4; ++s) xr[s] = fetch_x<T>(A, tok, (int64_t)t * TC + s * 32 + g4 * 8, mine);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int g = 0; g < SG; ++g) {
                const int gi = min((t * TC + g * (TC / SG)) / A.group, A.groups - 1);     // past the last column x is 0
                const int64_t at = ((int64_t)min(rt0 + i, A.row_tiles - 1) * A.groups + gi) * TR + g4 * 4;
                sc[i][g] = *(const t4 *)((const T *)A.scales + at);
                z[i][g] = ZEROS ? A.zeros[at / 4] : 0x08080808u;
            }
        if (t + waves < A.tiles) weights(t + waves, ahead);
        f32x4 c[RT], sx = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < RT; ++i) c[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const frag<M> xf = part_x<T>(xr[s], n % PARTS);
            sx = mma(one, xf, sx);
#pragma unroll
            for (int i = 0; i < RT; ++i) c[i] = mma(unpack<T>(s == 0 ? w[i].x : s == 1 ? w[i].y : s == 2 ? w[i].z : w[i].w), xf, c[i]);
            if ((s + 1) % (4 / SG) == 0) {
                const int g = s / (4 / SG);
#pragma unroll
                for (int i = 0; i < RT; ++i) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        y[i][r] += (float)sc[i][g][r] * (c[i][r] - (float)(16 + ((z[i][g] >> (8 * r)) & 255)) * sx[r]);
                    c[i] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
                sx = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
    }
    // the waves' sums in wave order, a row tile at a time
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        if (i) __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r) part[wave][g4 * 4 + r][n] = y[i][r];
        __syncthreads();
        for (int e = threadIdx.x; e < TR * PER; e += blockDim.x) {
            const int r = e % TR, t = e / TR;
            const int64_t row = (int64_t)(rt0 + i) * TR + r;
            if (row >= A.rows || t0 + t >= A.tokens) continue;
            float sum = 0.f;
            for (int wv = 0; wv < waves; ++wv)
#pragma unroll
                for (int p = 0; p < PARTS; ++p) sum += part[wv][r][t * PARTS + p];
            ((T *)A.y)[(t0 + t) * A.y_stride + row] = (T)sum;
        }
    }
}

struct LayoutArgs {
    const uint8_t *packed, *zeros;
    const void *scales;
    uint32_t *w;
    void *ls;
    uint8_t *lz;
    int64_t rows, cols, packed_stride, scale_stride, zero_stride, words, entries;
    int tiles, groups;
    bool words_aligned;
};

// Nibble j of 8 to place j / 2 + 4 (j % 2): the even ones to the low half, the odd ones to the high half.
__device__ __forceinline__ uint32_t pair_up(uint32_t x) {
    auto low = [](uint32_t v) {
        v &= 0x0f0f0f0fu;
        v = (v | v >> 4) & 0x00ff00ffu;
        return (v | v >> 8) & 0xffffu;
    };
    return low(x) | low(x >> 4) << 16;
}

template <typename T> __global__ __launch_bounds__(256) void layout_kernel(LayoutArgs A) {
    const int64_t step = (int64_t)gridDim.x * blockDim.x, i0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (int64_t i = i0; i < A.words / 4; i += step) {
        // word s of lane l of tile (rt, t): row l % 16, columns 128 t + 32 s + 8 (l / 16) + 0..7
        const int l = (int)(i & 63);
        const int64_t tile = i >> 6, rt = tile / A.tiles, t = tile - rt * A.tiles, row = rt * TR + (l & 15);
        uint32_t out[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int64_t c = t * TC + s * 32 + (l >> 4) * 8;
            uint32_t q = 0;
            if (row < A.rows && c < A.cols) {
                const uint8_t *p = A.packed + row * A.packed_stride + c / 2;
                if (A.words_aligned && c + 8 <= A.cols) {
                    q = *(const uint32_t *)p;
                } else {
                    for (int j = 0; j < 8 && c + j < A.cols; ++j) q |= (uint32_t)(p[j / 2] >> (4 * (j & 1)) & 15) << (4 * j);
                }
            }
            out[s] = pair_up(q);
        }
        ((uint4 *)A.w)[i] = make_uint4(out[0], out[1], out[2], out[3]);
    }
    for (int64_t i = i0; i < A.entries; i += step) {
        const int64_t r = i % TR, gi = i / TR % A.groups, row = i / TR / A.groups * TR + r;
        ((T *)A.ls)[i] = row < A.rows ? ((const T *)A.scales)[row * A.scale_stride + gi] : (T)0.f;
        if (A.lz) A.lz[i] = row < A.rows ? A.zeros[row * A.zero_stride + gi] : 0;
    }
}

// ------------------------------------------------------------------------------------------------ host
thread_local char g_detail[256] = "";
int fail(int status, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int status, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_detail, sizeof g_detail, fmt, ap);
    va_end(ap);
    return status;
}

struct Shape {
    int64_t row_tiles, tiles, groups, es, w_bytes, s_bytes, z_bytes, total;
};
int shape_of(const spmm_q4_desc_t *w, const char *where, Shape *s) {
    if (!w) return fail(SPMM_HIP_ERR_ARG, "%s: no description", where);
    if (w->dtype != SPMM_Q4_F32 && w->dtype != SPMM_Q4_F16 && w->dtype != SPMM_Q4_BF16)
        return fail(SPMM_HIP_ERR_ARG, "%s: element type %d", where, w->dtype);
    if (w->rows < 0 || w->cols < 0) return fail(SPMM_HIP_ERR_ARG, "%s: negative sizes", where);
    if (w->rows > (1 << 30) || w->cols > (1 << 30)) return fail(SPMM_HIP_ERR_OVERFLOW, "%s: more than 2^30 rows or columns", where);
    if (w->group != 32 && w->group != 64 && (w->group < 128 || w->group % 128))
        return fail(SPMM_HIP_ERR_ARG, "%s: groups of %d columns (32, 64 or a multiple of 128)", where, w->group);
    if (w->zeros < 0 || w->zeros > 1) return fail(SPMM_HIP_ERR_ARG, "%s: zeros = %d", where, w->zeros);
    s->row_tiles = (w->rows + TR - 1) / TR;
    s->tiles = (w->cols + TC - 1) / TC;
    s->groups = (w->cols + w->group - 1) / w->group;
    s->es = w->dtype == SPMM_Q4_F32 ? 4 : 2;
    auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
    s->w_bytes = s->row_tiles * s->tiles * 1024;
    s->s_bytes = up(s->row_tiles * s->groups * TR * s->es);
    s->z_bytes = w->zeros ? up(s->row_tiles * s->groups * TR) : 0;
    s->total = s->w_bytes + s->s_bytes + s->z_bytes;
    return SPMM_HIP_OK;
}

struct OnDevice {
    int prev = -1, status = SPMM_HIP_OK;
    OnDevice(int device, const char *where) {
        int n = 0;
        if (hipGetDeviceCount(&n) != hipSuccess || device < 0 || device >= n) {
            (void)hipGetLastError();
            status = fail(SPMM_HIP_ERR_NODEVICE, "%s: no HIP device %d", where, device);
            return;
        }
        hipError_t e = hipGetDevice(&prev);
        if (e == hipSuccess && prev != device) e = hipSetDevice(device);
        else if (e == hipSuccess) prev = -1;
        if (e != hipSuccess) {
            prev = -1;
            status = fail(SPMM_HIP_ERR_HIP, "%s: %s", where, hipGetErrorString(e));
        }
    }
    ~OnDevice() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
};

int launch(const void *kernel, const char *where, dim3 grid, int threads, void **args, void *stream) {
    const hipError_t e = hipLaunchKernel(kernel, grid, dim3((unsigned)threads), args, 0, (hipStream_t)stream);
    return e == hipSuccess ? SPMM_HIP_OK : fail(SPMM_HIP_ERR_HIP, "%s launch: %s", where, hipGetErrorString(e));
}

template <typename T, bool ZEROS, int RT> const void *matvec_sg(int group) {
    return group >= 128 ? (const void *)matvec_kernel<T, ZEROS, RT, 1>
           : group == 64 ? (const void *)matvec_kernel<T, ZEROS, RT, 2> : (const void *)matvec_kernel<T, ZEROS, RT, 4>;
}
template <typename T, bool ZEROS> const void *matvec_rt(int rt, int group) {
    return rt == 4 ? (const void *)matvec_kernel<T, ZEROS, 4, 1> : rt == 2 ? matvec_sg<T, ZEROS, 2>(group) : matvec_sg<T, ZEROS, 1>(group);
}
template <typename T> const void *matvec_of(bool zeros, int rt, int group) {
    return zeros ? matvec_rt<T, true>(rt, group) : matvec_rt<T, false>(rt, group);
}

}  // namespace

extern "C" {

const char *spmm_q4_last_error_detail(void) { return g_detail; }

int spmm_q4_layout_bytes(const spmm_q4_desc_t *w, size_t *bytes) {
    Shape s;
    const int st = shape_of(w, "q4_layout_bytes", &s);
    if (st != SPMM_HIP_OK) return st;
    if (!bytes) return fail(SPMM_HIP_ERR_ARG, "q4_layout_bytes: bytes is NULL");
    *bytes = (size_t)s.total;
    return SPMM_HIP_OK;
}

int spmm_q4_layout(const spmm_q4_desc_t *w, const void *packed, int64_t packed_stride, const void *scales,
                   int64_t scale_stride, const void *zeros, int64_t zero_stride, void *dst, size_t dst_bytes, void *stream) {
    const char *W = "q4_layout";
    Shape s;
    const int st = shape_of(w, W, &s);
    if (st != SPMM_HIP_OK) return st;
    if (s.total == 0) return SPMM_HIP_OK;
    if (!packed || !scales || (w->zeros && !zeros)) return fail(SPMM_HIP_ERR_ARG, "%s: packed, scales or zeros are NULL", W);
    if (!w->zeros && zeros) return fail(SPMM_HIP_ERR_ARG, "%s: zero points for a description without", W);
    if (packed_stride < 0 || scale_stride < 0 || zero_stride < 0) return fail(SPMM_HIP_ERR_ARG, "%s: negative strides", W);
    if ((uintptr_t)scales % s.es) return fail(SPMM_HIP_ERR_ARG, "%s: the scales are not aligned", W);
    if (!dst || (uintptr_t)dst % 256 || dst_bytes < (size_t)s.total)
        return fail(SPMM_HIP_ERR_ARG, "%s: the layout needs %lld bytes, 256-byte aligned", W, (long long)s.total);
    OnDevice on(w->device, W);
    if (on.status) return on.status;
    LayoutArgs A = {};
    A.packed = (const uint8_t *)packed;
    A.zeros = (const uint8_t *)zeros;
    A.scales = scales;
    A.w = (uint32_t *)dst;
    A.ls = (char *)dst + s.w_bytes;
    A.lz = w->zeros ? (uint8_t *)dst + s.w_bytes + s.s_bytes : nullptr;
    A.rows = w->rows;
    A.cols = w->cols;
    A.packed_stride = packed_stride;
    A.scale_stride = scale_stride;
    A.zero_stride = zero_stride;
    A.words = s.w_bytes / 4;
    A.entries = s.row_tiles * s.groups * TR;
    A.tiles = (int)s.tiles;
    A.groups = (int)s.groups;
    A.words_aligned = (uintptr_t)packed % 4 == 0 && packed_stride % 4 == 0;
    const int64_t blocks = (A.words / 4 + 255) / 256;
    void *args[] = {&A};
    return launch(s.es == 4 ? (const void *)layout_kernel<float> : (const void *)layout_kernel<uint16_t>, W,
                  dim3((unsigned)(blocks < 8192 ? blocks : 8192)), 256, args, stream);
}

int spmm_q4_matvec(const spmm_q4_desc_t *w, const void *layout, const void *x, int64_t x_stride, int64_t tokens, void *y,
                   int64_t y_stride, void *stream) {
    const char *W = "q4_matvec";
    Shape s;
    const int st = shape_of(w, W, &s);
    if (st != SPMM_HIP_OK) return st;
    if (tokens < 0 || x_stride < 0 || y_stride < 0) return fail(SPMM_HIP_ERR_ARG, "%s: negative sizes or strides", W);
    if (tokens > 65535) return fail(SPMM_HIP_ERR_OVERFLOW, "%s: %lld vectors", W, (long long)tokens);
    if (tokens == 0 || w->rows == 0) return SPMM_HIP_OK;
    if (!y || (uintptr_t)y % s.es || (tokens > 1 && y_stride < w->rows))
        return fail(SPMM_HIP_ERR_ARG, "%s: y is NULL, not aligned, or its rows overlap", W);
    if (w->cols > 0 && (!layout || (uintptr_t)layout % 256 || !x || (uintptr_t)x % s.es))
        return fail(SPMM_HIP_ERR_ARG, "%s: the layout or x is NULL or not aligned", W);
    OnDevice on(w->device, W);
    if (on.status) return on.status;
    Args A = {};
    A.w = (const uint4 *)layout;
    A.scales = (const char *)layout + s.w_bytes;
    A.zeros = w->zeros ? (const uint32_t *)((const char *)layout + s.w_bytes + s.s_bytes) : nullptr;
    A.x = (const char *)x;
    A.y = (char *)y;
    A.rows = w->rows;
    A.cols = w->cols;
    A.x_stride = x_stride;
    A.y_stride = y_stride;
    A.tokens = tokens;
    A.tiles = (int)s.tiles;
    A.groups = (int)s.groups;
    A.row_tiles = (int)s.row_tiles;
    A.group = w->group;
    A.wide = (uintptr_t)x % 16 == 0 && (tokens == 1 || x_stride % (16 / s.es) == 0);
    // Row tiles that share a block's x: as many as leave a block for every compute unit.  Waves that share the columns: 16 a
    // compute unit in all, one column tile each at least.  Four vectors in bf16 with 1, 2 and 4 row tiles: 4096 x 4096 weights
    // 5.8, 7.0, 10.2 us, 8192 x 8192 16.1, 12.6, 17.0, 32768 x 4096 28.6, 20.0, 18.0; 16384 x 4096 with 1024, 2048, 4096 and
    // 8192 waves 24.1, 15.7, 12.1, 14.0.  Four only where a tile has one scale a row: with more the registers do not hold
    // them.  32768 x 4096, four vectors, two and four row tiles: groups of 128 in bf16 17.7, 16.3, fp16 17.6, 16.4, fp32 42.4,
    // 33.6; of 64 19.5, 20.1, 19.2, 21.7, 44.7, 52.3; of 32 24.5, 32.8, 22.8, 35.1, 47.5, 105.9.
    const int rt = s.row_tiles >= 8 * 256 && w->group >= 128 ? 4 : s.row_tiles >= 2 * 256 ? 2 : 1;
    const int64_t blocks = (s.row_tiles + rt - 1) / rt;
    int waves = 1;
    while (waves < WMAX && waves < A.tiles && blocks * waves < 4096) waves *= 2;
    const int per = w->dtype == SPMM_Q4_F32 ? 5 : 16;
    void *args[] = {&A};
    const void *kern = w->dtype == SPMM_Q4_F32 ? matvec_of<float>(w->zeros, rt, w->group)
                       : w->dtype == SPMM_Q4_F16 ? matvec_of<_Float16>(w->zeros, rt, w->group)
                                                 : matvec_of<__bf16>(w->zeros, rt, w->group);
    return launch(kern, W, dim3((unsigned)blocks, (unsigned)((tokens + per - 1) / per)), waves * 64, args, stream);
}

}  // extern "C"
