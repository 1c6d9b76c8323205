// attn_host.hip -- the checks and launches that the attention operators share on the host (include/spmm_attn.h).
#include "attn_common.hpp"

namespace attn {

thread_local char g_detail[256] = "";

int fail(int status, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_detail, sizeof g_detail, fmt, ap);
    va_end(ap);
    return status;
}

size_t elem_size(int dtype) { return dtype == SPMM_ATTN_F32 ? 4 : 2; }

int check_desc(const spmm_attn_desc_t *a, const char *where) {
    if (!a) return fail(SPMM_HIP_ERR_ARG, "%s: no description", where);
    if (a->dtype != SPMM_ATTN_F32 && a->dtype != SPMM_ATTN_F16 && a->dtype != SPMM_ATTN_BF16)
        return fail(SPMM_HIP_ERR_ARG, "%s: element type %d", where, a->dtype);
    if (a->kv_heads < 1 || a->heads < 1 || a->heads % a->kv_heads || a->heads > 65535)
        return fail(SPMM_HIP_ERR_ARG, "%s: %d heads over %d key heads", where, a->heads, a->kv_heads);
    if (a->dim < 1 || a->dim > SPMM_ATTN_MAX_DIM)
        return fail(SPMM_HIP_ERR_ARG, "%s: head width %d is not in 1 .. %d", where, a->dim, SPMM_ATTN_MAX_DIM);
    if (a->window < 0 || a->sinks < 0)
        return fail(SPMM_HIP_ERR_ARG, "%s: window %d, sinks %d", where, a->window, a->sinks);
    if (!std::isfinite(a->scale * LOG2E))            // what the kernels use
        return fail(SPMM_HIP_ERR_ARG, "%s: the scale %g, times log2(e), is not finite", where, a->scale);
    if (a->zero_rest < 0 || a->zero_rest > 1 || a->reserved != 0)
        return fail(SPMM_HIP_ERR_ARG, "%s: zero_rest %d, reserved %d", where, a->zero_rest, a->reserved);
    if (a->batch < 0 || a->q_len < 0 || a->k_len < 0)
        return fail(SPMM_HIP_ERR_ARG, "%s: negative sizes", where);
    if (a->batch > INT32_MAX / 2 || a->q_len > INT32_MAX / 2 || a->k_len > INT32_MAX / 2)
        return fail(SPMM_HIP_ERR_OVERFLOW, "%s: more than 2^30 sequences or rows", where);
    return SPMM_HIP_OK;
}

int check_rows(const spmm_attn_desc_t *a, const spmm_attn_rows_t *r, const char *where, const char *name, int64_t batch,
               int64_t rows, int heads, bool written, Rows *out) {
    if (!r) return fail(SPMM_HIP_ERR_ARG, "%s: %s is missing", where, name);
    const size_t es = elem_size(a->dtype);
    if (batch > 0 && rows > 0) {
        if (!r->ptr) return fail(SPMM_HIP_ERR_ARG, "%s: %s is NULL", where, name);
        if ((uintptr_t)r->ptr % es) return fail(SPMM_HIP_ERR_ARG, "%s: %s is not aligned to its elements", where, name);
    }
    // strides in order of size, each at least what the smaller ones span
    struct { int64_t stride, count; } d[3] = {{r->seq, batch}, {r->row, rows}, {r->head, (int64_t)heads}};
    const int64_t lim = INT64_C(1) << 60;
    for (auto &x : d) {
        const int64_t m = x.stride < 0 ? -(x.stride + 1) : x.stride;
        if (x.count > 1 && m > lim / x.count)
            return fail(SPMM_HIP_ERR_OVERFLOW, "%s: the strides of %s pass 2^60", where, name);
        if (x.count > 1 && x.stride < 0) return fail(SPMM_HIP_ERR_ARG, "%s: a stride of %s is negative", where, name);
    }
    if (written && batch > 0 && rows > 0) {
        int64_t span = a->dim;
        bool used[3] = {};
        for (int i = 0; i < 3; ++i) {
            int best = -1;
            for (int j = 0; j < 3; ++j)
                if (!used[j] && d[j].count > 1 && (best < 0 || d[j].stride < d[best].stride)) best = j;
            if (best < 0) break;
            used[best] = true;
            if (d[best].stride < span) return fail(SPMM_HIP_ERR_ARG, "%s: rows of %s overlap", where, name);
            span = d[best].stride * (d[best].count - 1) + span;
        }
    }
    out->ptr = (char *)r->ptr;
    out->seq = r->seq;
    out->row = r->row;
    out->head = r->head;
    // reads in 16-byte pieces; writes in 4 elements
    const int64_t el = written ? 4 : 16 / (int64_t)es;
    out->wide = (uintptr_t)r->ptr % (el * es) == 0 && a->dim % el == 0;
    for (auto &x : d)
        if (x.count > 1 && x.stride % el) out->wide = false;
    out->direct = out->wide && r->row >= a->dim && r->row < INT32_MAX / 128 / (int64_t)es;
    return SPMM_HIP_OK;
}

int launch(const void *kernel, const char *where, int64_t blocks, int threads, void **args, void *stream) {
    if (blocks <= 0) return SPMM_HIP_OK;
    if (blocks > INT32_MAX) return fail(SPMM_HIP_ERR_OVERFLOW, "%s: %lld blocks", where, (long long)blocks);
    const hipError_t e = hipLaunchKernel(kernel, dim3((unsigned)blocks), dim3((unsigned)threads), args, 0,
                                         (hipStream_t)stream);
    return e == hipSuccess ? SPMM_HIP_OK : fail(SPMM_HIP_ERR_HIP, "%s launch: %s", where, hipGetErrorString(e));
}

OnDevice::OnDevice(int device, const char *where) {
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
OnDevice::~OnDevice() {
    if (prev >= 0) (void)hipSetDevice(prev);
}

}  // namespace attn

extern "C" const char *spmm_attn_last_error_detail(void) { return attn::g_detail; }
