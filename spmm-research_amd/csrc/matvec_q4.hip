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

// 8 elements of part `part` of x[tok][k ...]
template <typename T> __device__ __forceinline__ frag<typename Kind<T>::M> load_x(const Args &A, int64_t tok, int part, int64_t k, bool mine) {
    using M = typename Kind<T>::M;
    frag<M> f = {};
    if (!mine || k >= A.cols) return f;
    const T *p = (const T *)A.x + tok * A.x_stride + k;
    T e[8];
    if (A.wide && k + 8 <= A.cols) {
        __builtin_memcpy(e, __builtin_assume_aligned(p, 16), sizeof e);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = k + j < A.cols ? p[j] : (T)0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (sizeof(T) == 2) {
            f[j] = e[j];
        } else {
            // 8 bits of the value at a time, cut off, so each rest is exact; an infinity or NaN is all in the first part
            float r = e[j];
            uint32_t hi = __builtin_bit_cast(uint32_t, r) & 0xffff0000u;
            for (int i = 0; i < part; ++i) {
                r = (hi & 0x7f800000u) == 0x7f800000u ? 0.f : r - __builtin_bit_cast(float, hi);
                hi = __builtin_bit_cast(uint32_t, r) & 0xffff0000u;
            }
            if (part == 0 && r != r) hi |= 0x00400000u;
            f[j] = __builtin_bit_cast(__bf16, (uint16_t)(hi >> 16));
        }
    }
    return f;
}

template <typename T, bool ZEROS> __global__ void matvec_kernel(Args A) {
    using K = Kind<T>;
    using M = typename K::M;
    constexpr int PARTS = K::PARTS, PER = 16 / PARTS;        // vectors a block takes
    __shared__ float part[WMAX][TR][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, n = lane & 15, g4 = lane >> 4;
    const int rt = blockIdx.x;
    const int64_t t0 = (int64_t)blockIdx.y * PER, tok = t0 + n / PARTS;
    const bool mine = n < PER * PARTS && tok < A.tokens;
    const uint4 *w = A.w + (int64_t)rt * A.tiles * 64 + lane;
    frag<M> one;
#pragma unroll
    for (int j = 0; j < 8; ++j) one[j] = (M)1.f;

    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    const int steps = A.group < TC ? A.group / 32 : 4;       // products of a scale
    uint4 next = wave < A.tiles ? w[(int64_t)wave * 64] : make_uint4(0, 0, 0, 0);
    for (int t = wave; t < A.tiles; t += waves) {
        const uint4 now = next;
        if (t + waves < A.tiles) next = w[(int64_t)(t + waves) * 64];
        const uint32_t word[4] = {now.x, now.y, now.z, now.w};
        f32x4 c = {0.f, 0.f, 0.f, 0.f}, sx = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int64_t k = (int64_t)t * TC + s * 32;
            const frag<M> xf = load_x<T>(A, tok, n % PARTS, k + g4 * 8, mine);
            c = mma(unpack<T>(word[s]), xf, c);
            sx = mma(one, xf, sx);
            if ((s + 1) % steps == 0) {
                const int64_t gi = k / A.group;
                if (gi < A.groups) {
                    const int64_t at = ((int64_t)rt * A.groups + gi) * TR + g4 * 4;
                    typedef T t4 __attribute__((ext_vector_type(4)));
                    const t4 sc = *(const t4 *)((const T *)A.scales + at);
                    const uint32_t z4 = ZEROS ? A.zeros[at / 4] : 0x08080808u;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        y[r] += (float)sc[r] * (c[r] - (float)(16 + ((z4 >> (8 * r)) & 255)) * sx[r]);
                }
                c = sx = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][g4 * 4 + r][n] = y[r];
    __syncthreads();
    for (int i = threadIdx.x; i < TR * PER; i += blockDim.x) {
        const int r = i % TR, t = i / TR;
        const int64_t row = (int64_t)rt * TR + r;
        if (row >= A.rows || t0 + t >= A.tokens) continue;
        float sum = 0.f;
        for (int wv = 0; wv < waves; ++wv)
#pragma unroll
            for (int p = 0; p < PARTS; ++p) sum += part[wv][r][t * PARTS + p];
        ((T *)A.y)[(t0 + t) * A.y_stride + row] = (T)sum;
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
};

template <typename T> __global__ __launch_bounds__(256) void layout_kernel(LayoutArgs A) {
    const int64_t step = (int64_t)gridDim.x * blockDim.x, i0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (int64_t i = i0; i < A.words; i += step) {
        // word s of lane l of tile (rt, t): row l % 16, columns 128 t + 32 s + 8 (l / 16) + 0..7
        const int s = (int)(i & 3), l = (int)((i >> 2) & 63);
        const int64_t tile = i >> 8, rt = tile / A.tiles, t = tile % A.tiles, row = rt * TR + (l & 15);
        const int64_t c0 = t * TC + s * 32 + (l >> 4) * 8;
        uint32_t out = 0;
        for (int j = 0; j < 8; ++j) {
            const int64_t c = c0 + j;
            uint32_t q = 0;
            if (row < A.rows && c < A.cols) q = (A.packed[row * A.packed_stride + c / 2] >> (4 * (c & 1))) & 15u;
            out |= q << (4 * ((j >> 1) + 4 * (j & 1)));
        }
        A.w[i] = out;
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

template <typename T> const void *matvec_of(bool zeros) {
    return zeros ? (const void *)matvec_kernel<T, true> : (const void *)matvec_kernel<T, false>;
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
    const int64_t blocks = (A.words + 255) / 256;
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
    // waves share a row tile's columns: about 16 waves a compute unit in all, one column tile each at least
    int waves = 1;
    while (waves < WMAX && waves < A.tiles && s.row_tiles * waves < 4096) waves *= 2;
    const int per = w->dtype == SPMM_Q4_F32 ? 5 : 16;
    void *args[] = {&A};
    const void *kern = w->dtype == SPMM_Q4_F32 ? matvec_of<float>(w->zeros)
                       : w->dtype == SPMM_Q4_F16 ? matvec_of<_Float16>(w->zeros) : matvec_of<__bf16>(w->zeros);
    return launch(kern, W, dim3((unsigned)s.row_tiles, (unsigned)((tokens + per - 1) / per)), waves * 64, args, stream);
}

}  // extern "C"
