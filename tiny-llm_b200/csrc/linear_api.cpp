// Entry points of the W8A16 projections (include/tllm_kv.h): argument checks
// and the choice of the kernel. No handle and no workspace: the calls run on
// the current device, on the caller's stream, and read errors back with
// tl_last_error(NULL).
#include <cstdint>
#include <cuda_runtime.h>

#include "kernels.h"
#include "linear_pack.cuh"
#include "paged_kv.h"
#include "tllm_kv.h"

using tllm::set_thread_error;

namespace {

constexpr int kMaxRows = 1 << 20, kMaxK = 1 << 20, kMaxN = 1 << 22;

bool misaligned(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

// TL_OK, or the refusal of a weight's shape.
int check_shape(const char *ctx, int k, int n, int group_size) {
    if (k <= 0 || n <= 0) return set_thread_error(TL_ERR_INVALID_ARG, "%s: k and n must be positive", ctx);
    if (group_size != 32 && group_size != 64 && group_size != 128)
        return set_thread_error(TL_ERR_UNSUPPORTED, "%s: group_size must be 32, 64 or 128", ctx);
    if (k > kMaxK || n > kMaxN)
        return set_thread_error(TL_ERR_UNSUPPORTED, "%s: k above 2^20 or n above 2^22 is not supported", ctx);
    return TL_OK;
}

int linear(const char *ctx, tllm::LinearArgs a, cudaStream_t stream) {
    if (int st = check_shape(ctx, a.k, a.n, a.group)) return st;
    if (a.act < TL_ACT_NONE || a.act > TL_ACT_SILU)
        return set_thread_error(TL_ERR_INVALID_ARG, "%s: unknown activation %d", ctx, a.act);
    if (a.rows < 0) return set_thread_error(TL_ERR_INVALID_ARG, "%s: rows must be >= 0", ctx);
    if (a.rows > kMaxRows) return set_thread_error(TL_ERR_UNSUPPORTED, "%s: more than 2^20 rows are not supported", ctx);
    if (a.rows == 0) return TL_OK;
    if (!a.x || !a.y) return set_thread_error(TL_ERR_INVALID_ARG, !a.x ? "%s: input is null" : "%s: output is null", ctx);
    if (!a.packed) return set_thread_error(TL_ERR_INVALID_ARG, "%s: packed weights are null", ctx);
    if (misaligned(a.x, 16) || misaligned(a.packed, 16))
        return set_thread_error(TL_ERR_INVALID_ARG, "%s: input and packed weights must be 16-byte aligned", ctx);
    if (misaligned(a.y, 2) || misaligned(a.bias, 2) || misaligned(a.bias2, 2) || misaligned(a.residual, 2))
        return set_thread_error(TL_ERR_INVALID_ARG, "%s: a pointer is not aligned to its elements", ctx);
    if (a.rows == 1) {  // no stride is used
        a.x_stride = (a.k + 7) / 8 * 8;
        a.y_stride = a.residual_stride = a.n;
    }
    if (a.x_stride < a.k || a.x_stride % 8 != 0)
        return set_thread_error(TL_ERR_INVALID_ARG, "%s: x_stride must be at least k and a multiple of 8", ctx);
    if (a.y_stride < a.n || (a.residual && a.residual_stride < a.n))
        return set_thread_error(TL_ERR_INVALID_ARG, "%s: the strides of output and residual must be at least n", ctx);
    if (a.residual == a.y && a.residual_stride != a.y_stride)
        return set_thread_error(TL_ERR_INVALID_ARG, "%s: a residual in place needs the output's stride", ctx);
    const int sms = tllm::current_device_sms();
    if (sms == 0) return set_thread_error(TL_ERR_NO_DEVICE, "%s: no CUDA device", ctx);
    const cudaError_t e = a.rows <= tllm::kLinearFewRows ? tllm::launch_linear(a, sms, stream)
                                                         : tllm::launch_linear_tc(a, sms, stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_thread_error(TL_ERR_CUDA, "%s: launch failed: %s", ctx, cudaGetErrorString(e));
    }
    return TL_OK;
}

}  // namespace

extern "C" {

size_t tl_linear_packed_bytes(int k, int n, int group_size, int gated) {
    if (check_shape("linearPackedBytes", k, n, group_size) != TL_OK) return 0;
    return (size_t)tllm::lin::tiles(n, gated != 0) * (size_t)tllm::lin::blocks(k) *
           (size_t)tllm::lin::unit_bytes(group_size);
}

int tl_linear_pack(const int8_t *w, const void *scales, const int8_t *w_up, const void *scales_up, int k, int n,
                   int group_size, void *packed, tl_stream_t stream) {
    const char *ctx = "linearPack";
    if (int st = check_shape(ctx, k, n, group_size)) return st;
    if (!w || !scales || !packed) return set_thread_error(TL_ERR_INVALID_ARG, "%s: a weight or scale pointer is null", ctx);
    if (!w_up != !scales_up)
        return set_thread_error(TL_ERR_INVALID_ARG, "%s: a gated pair needs w_up and scales_up both", ctx);
    if (misaligned(packed, 16) || misaligned(scales, 2) || misaligned(scales_up, 2))
        return set_thread_error(TL_ERR_INVALID_ARG, "%s: packed must be 16-byte and scales 2-byte aligned", ctx);
    const uintptr_t p0 = reinterpret_cast<uintptr_t>(packed), p1 = p0 + tl_linear_packed_bytes(k, n, group_size, w_up != nullptr);
    const uintptr_t wb = (uintptr_t)k * (uintptr_t)n, sb = (uintptr_t)((k + group_size - 1) / group_size) * (uintptr_t)n * 2;
    auto hits = [&](const void *q, uintptr_t bytes) {
        const uintptr_t q0 = reinterpret_cast<uintptr_t>(q);
        return q && q0 < p1 && p0 < q0 + bytes;
    };
    if (hits(w, wb) || hits(w_up, wb) || hits(scales, sb) || hits(scales_up, sb))
        return set_thread_error(TL_ERR_INVALID_ARG, "%s: source and destination overlap", ctx);
    const int sms = tllm::current_device_sms();
    if (sms == 0) return set_thread_error(TL_ERR_NO_DEVICE, "%s: no CUDA device", ctx);
    const cudaError_t e =
        tllm::launch_linear_pack(w, scales, w_up, scales_up, k, n, group_size, packed, sms, (cudaStream_t)stream);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_thread_error(TL_ERR_CUDA, "%s: launch failed: %s", ctx, cudaGetErrorString(e));
    }
    return TL_OK;
}

int tl_linear(const void *x, long long x_stride, int rows, const void *packed, int k, int n, int group_size,
              const void *bias, int activation, const void *residual, long long residual_stride, void *y,
              long long y_stride, tl_stream_t stream) {
    tllm::LinearArgs a{};
    a.x = x;
    a.x_stride = x_stride;
    a.packed = packed;
    a.rows = rows;
    a.k = k;
    a.n = n;
    a.group = group_size;
    a.act = activation;
    a.bias = bias;
    a.residual = residual;
    a.residual_stride = residual_stride;
    a.y = y;
    a.y_stride = y_stride;
    return linear("linear", a, (cudaStream_t)stream);
}

int tl_linear_gated(const void *x, long long x_stride, int rows, const void *packed, int k, int n, int group_size,
                    const void *bias, const void *bias_up, int activation, void *y, long long y_stride,
                    tl_stream_t stream) {
    tllm::LinearArgs a{};
    a.x = x;
    a.x_stride = x_stride;
    a.packed = packed;
    a.rows = rows;
    a.k = k;
    a.n = n;
    a.group = group_size;
    a.gated = 1;
    a.act = activation;
    a.bias = bias;
    a.bias2 = bias_up;
    a.y = y;
    a.y_stride = y_stride;
    return linear("linearGated", a, (cudaStream_t)stream);
}

}  // extern "C"
