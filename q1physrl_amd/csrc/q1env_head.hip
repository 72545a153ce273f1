// q1env_head.hip - the wide categorical head of libq1env.so (include/q1env.h q1env_head_*): log-probability, entropy and cross entropy of given
// classes from hidden rows and the head's weights without the logits ever being kept, and the gradients (kernels: q1head.hpp, what runs when: q1head_calls.hpp).
#include "q1head_calls.hpp"

using namespace q1head;

namespace {

int check_shape(const char* who, int dtype, int64_t rows, int64_t width, int64_t classes) {
    if (dtype != Q1ENV_DT_F32 && dtype != Q1ENV_DT_BF16 && dtype != Q1ENV_DT_F16) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": unknown dtype");
    if (rows < 0 || rows > MAX_ROWS) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": rows out of range (0 .. 2^22)");
    if (width < 1 || width > MAX_WIDTH) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": width out of range (1 .. 2^16)");
    if (classes < 1 || classes > MAX_CLASSES) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": classes out of range (1 .. 2^22)");
    return 0;
}

int check_head(const char* who, const q1env_head* hd) {
    if (!hd) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": null argument");
    if (int rc = check_shape(who, hd->dtype, hd->rows, hd->width, hd->classes)) return rc;
    if (!hd->weight_dev || (hd->rows > 0 && !hd->hidden_dev)) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": hidden / weight is NULL");
    if (hd->hidden_stride < hd->width || hd->weight_stride < hd->width) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": a row stride is smaller than the width");
    const uintptr_t size = elem_size(hd->dtype);
    if ((uintptr_t)hd->hidden_dev % size || (uintptr_t)hd->weight_dev % size || (uintptr_t)hd->bias_dev % size)
        return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": a pointer is not aligned to its element size");
    if (hd->rows > 0 && !hd->state_dev) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": state is NULL");
    return 0;
}

int guard_device(const char* who, int device) {
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n == 0) return fail(Q1ENV_ERR_NO_DEVICE, std::string(who) + ": no HIP device (there is no CPU fallback)");
    if (device < 0 || device >= n) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": no such device");
    return 0;
}

}  // namespace

// zeros of a strided (rows, width) result, for a call without rows
static __global__ void __launch_bounds__(256) zero_rows_kernel(uint8_t* out, int64_t rows, int64_t row_bytes, int64_t stride_bytes) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * row_bytes; i += (int64_t)gridDim.x * 256) out[i / row_bytes * stride_bytes + i % row_bytes] = 0;
}

extern "C" {

uint64_t q1env_head_state_bytes(int64_t rows) { return rows < 0 || rows > MAX_ROWS ? 0 : State::bytes(rows); }

uint64_t q1env_head_workspace_bytes(int dtype, int64_t rows, int64_t width, int64_t classes, int backward) {
    if (check_shape("q1env_head_workspace_bytes", dtype, rows, width, classes)) return 0;
    if (rows == 0) return 256;
    return workspace_of(dtype, rows, width, classes, backward != 0);
}

int q1env_head_forward(int device, void* stream, const q1env_head* hd, int reduction, float* logp, float* entropy, float* loss) {
    const char* who = "q1env_head_forward";
    if (int rc = check_head(who, hd)) return rc;
    if (hd->target_bits != 32 && hd->target_bits != 64) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_forward: target_bits must be 32 or 64");
    if (hd->rows > 0 && (!hd->target_dev || !logp)) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_forward: target / logp is NULL");
    if (loss && !hd->state_dev) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_forward: state is NULL");
    if (reduction != Q1ENV_REDUCE_MEAN && reduction != Q1ENV_REDUCE_SUM) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_forward: unknown reduction");
    if (hd->rows > 0 && (!hd->ws_dev || hd->ws_bytes < q1env_head_workspace_bytes(hd->dtype, hd->rows, hd->width, hd->classes, 0)))
        return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_forward: workspace smaller than q1env_head_workspace_bytes(..., 0)");
    if (int rc = guard_device(who, device)) return rc;
    DeviceGuard guard(device);
    switch (hd->dtype) {
        case Q1ENV_DT_F32: return q1_head_forward_f32(device, (hipStream_t)stream, *hd, reduction, logp, entropy, loss);
        case Q1ENV_DT_BF16: return q1_head_forward_bf16(device, (hipStream_t)stream, *hd, reduction, logp, entropy, loss);
        default: return q1_head_forward_f16(device, (hipStream_t)stream, *hd, reduction, logp, entropy, loss);
    }
}

int q1env_head_backward(int device, void* stream, const q1env_head* hd, const float* dlogp, const float* dentropy, const float* dloss, void* dhidden, int64_t dhidden_stride,
                        void* dweight, int64_t dweight_stride, void* dbias) {
    const char* who = "q1env_head_backward";
    if (int rc = check_head(who, hd)) return rc;
    if (dloss && (dlogp || dentropy)) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: either dloss or the per-row gradients");
    if (!dloss && !dlogp && !dentropy) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: no upstream gradient");
    if (!dhidden && !dweight && !dbias) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: no result asked for");
    if ((dhidden && dhidden_stride < hd->width) || (dweight && dweight_stride < hd->width)) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: a row stride is smaller than the width");
    const uintptr_t size = elem_size(hd->dtype);
    if ((uintptr_t)dhidden % size || (uintptr_t)dweight % size || (uintptr_t)dbias % size) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: a pointer is not aligned to its element size");
    if (hd->rows > 0 && (!hd->ws_dev || hd->ws_bytes < q1env_head_workspace_bytes(hd->dtype, hd->rows, hd->width, hd->classes, 1)))
        return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: workspace smaller than q1env_head_workspace_bytes(..., 1)");
    if (int rc = guard_device(who, device)) return rc;
    DeviceGuard guard(device);
    if (hd->rows == 0) {                             // no sample: the weights' gradients are zero
        const int64_t es = (int64_t)elem_size(hd->dtype);
        if (dweight) hipLaunchKernelGGL(zero_rows_kernel, dim3(1024), dim3(256), 0, (hipStream_t)stream, (uint8_t*)dweight, hd->classes, hd->width * es, dweight_stride * es);
        if (dbias) hipLaunchKernelGGL(zero_rows_kernel, dim3(256), dim3(256), 0, (hipStream_t)stream, (uint8_t*)dbias, (int64_t)1, hd->classes * es, hd->classes * es);
        HIP_TRY(hipGetLastError());
        return Q1ENV_OK;
    }
    switch (hd->dtype) {
        case Q1ENV_DT_F32: return q1_head_backward_f32(device, (hipStream_t)stream, *hd, dlogp, dentropy, dloss, dhidden, dhidden_stride, dweight, dweight_stride, dbias);
        case Q1ENV_DT_BF16: return q1_head_backward_bf16(device, (hipStream_t)stream, *hd, dlogp, dentropy, dloss, dhidden, dhidden_stride, dweight, dweight_stride, dbias);
        default: return q1_head_backward_f16(device, (hipStream_t)stream, *hd, dlogp, dentropy, dloss, dhidden, dhidden_stride, dweight, dweight_stride, dbias);
    }
}

}  // extern "C"
