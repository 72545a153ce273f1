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
    if ((uintptr_t)hd->state_dev % 16 || (uintptr_t)hd->ws_dev % 16) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": state / workspace is not aligned to 16 bytes");
    if (hd->rows > 0 && !hd->state_dev) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": state is NULL");
    return 0;
}

// what the call writes - results, the workspace, the forward call's state - against everything that is read and each other
int check_apart(const char* who, const Extent* results, int n, const q1env_head& hd, uint64_t ws_bytes, bool backward) {
    const uintptr_t es = elem_size(hd.dtype);
    const Extent others[] = {{(uintptr_t)hd.hidden_dev, hd.rows, (uintptr_t)hd.width * es, (uintptr_t)hd.hidden_stride * es},
                             {(uintptr_t)hd.weight_dev, hd.classes, (uintptr_t)hd.width * es, (uintptr_t)hd.weight_stride * es},
                             {(uintptr_t)hd.bias_dev, 1, (uintptr_t)hd.classes * es, 0},
                             {backward ? 0 : (uintptr_t)hd.target_dev, 1, (uintptr_t)hd.rows * hd.target_bits / 8, 0},
                             {(uintptr_t)hd.state_dev, 1, q1env_head_state_bytes(hd.rows), 0},
                             {(uintptr_t)hd.ws_dev, 1, ws_bytes, 0}};
    for (int i = 0; i < n; ++i) {
        for (const Extent& o : others)
            if (!apart(results[i], o)) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": a result overlaps an operand, the state or the workspace");
        for (int k = 0; k < i; ++k)
            if (!apart(results[i], results[k])) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": two results overlap");
    }
    for (int k = 0; k < 4; ++k)
        if (!apart(others[k], others[5]) || (!backward && !apart(others[k], others[4])))
            return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": the state or the workspace overlaps an operand");
    return apart(others[4], others[5]) ? 0 : fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": the state overlaps the workspace");
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

}  // extern "C"

static int head_forward(int device, void* stream, const q1env_head* hd, int reduction, float* logp, float* entropy, float* loss) {
    const char* who = "q1env_head_forward";
    if (int rc = check_head(who, hd)) return rc;
    if (hd->target_bits != 32 && hd->target_bits != 64) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_forward: target_bits must be 32 or 64");
    if (hd->rows > 0 && (!hd->target_dev || !logp)) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_forward: target / logp is NULL");
    if (loss && !hd->state_dev) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_forward: state is NULL");
    if (reduction != Q1ENV_REDUCE_MEAN && reduction != Q1ENV_REDUCE_SUM) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_forward: unknown reduction");
    const uint64_t need = hd->rows > 0 ? q1env_head_workspace_bytes(hd->dtype, hd->rows, hd->width, hd->classes, 0) : 0;
    if (need && (!hd->ws_dev || hd->ws_bytes < need))
        return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_forward: workspace smaller than q1env_head_workspace_bytes(..., 0)");
    if ((uintptr_t)logp % 4 || (uintptr_t)entropy % 4 || (uintptr_t)loss % 4 || (uintptr_t)hd->target_dev % (hd->target_bits / 8)) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_forward: a pointer is not aligned to its element size");
    const Extent results[] = {{(uintptr_t)logp, 1, 4 * (uintptr_t)hd->rows, 0}, {(uintptr_t)entropy, 1, 4 * (uintptr_t)hd->rows, 0}, {(uintptr_t)loss, 1, 4, 0}};
    if (int rc = check_apart(who, results, 3, *hd, need, false)) return rc;
    if (int rc = guard_device(who, device)) return rc;
    DeviceGuard guard(device);
    switch (hd->dtype) {
        case Q1ENV_DT_F32: return q1_head_forward_f32(device, (hipStream_t)stream, *hd, reduction, logp, entropy, loss);
        case Q1ENV_DT_BF16: return q1_head_forward_bf16(device, (hipStream_t)stream, *hd, reduction, logp, entropy, loss);
        default: return q1_head_forward_f16(device, (hipStream_t)stream, *hd, reduction, logp, entropy, loss);
    }
}

static int head_backward(int device, void* stream, const q1env_head* hd, const float* dlogp, const float* dentropy, const float* dloss, void* dhidden, int64_t dhidden_stride, void* dweight,
                         int64_t dweight_stride, void* dbias) {
    const char* who = "q1env_head_backward";
    if (int rc = check_head(who, hd)) return rc;
    if (dloss && (dlogp || dentropy)) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: either dloss or the per-row gradients");
    if (!dloss && !dlogp && !dentropy) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: no upstream gradient");
    if (!dhidden && !dweight && !dbias) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: no result asked for");
    if ((dhidden && dhidden_stride < hd->width) || (dweight && dweight_stride < hd->width)) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: a row stride is smaller than the width");
    const uintptr_t size = elem_size(hd->dtype);
    if ((uintptr_t)dhidden % size || (uintptr_t)dweight % size || (uintptr_t)dbias % size) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: a pointer is not aligned to its element size");
    const uint64_t need = hd->rows > 0 ? q1env_head_workspace_bytes(hd->dtype, hd->rows, hd->width, hd->classes, 1) : 0;
    if (need && (!hd->ws_dev || hd->ws_bytes < need))
        return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: workspace smaller than q1env_head_workspace_bytes(..., 1)");
    if ((uintptr_t)dlogp % 4 || (uintptr_t)dentropy % 4 || (uintptr_t)dloss % 4) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: a pointer is not aligned to its element size");
    const Extent results[] = {{(uintptr_t)dhidden, hd->rows, hd->width * size, dhidden_stride * size}, {(uintptr_t)dweight, hd->classes, hd->width * size, dweight_stride * size},
                              {(uintptr_t)dbias, 1, hd->classes * size, 0}};
    if (int rc = check_apart(who, results, 3, *hd, need, true)) return rc;
    const Extent upstream[] = {{(uintptr_t)dlogp, 1, 4 * (uintptr_t)hd->rows, 0}, {(uintptr_t)dentropy, 1, 4 * (uintptr_t)hd->rows, 0}, {(uintptr_t)dloss, 1, 4, 0}};
    for (const Extent& u : upstream) {
        for (const Extent& r : results)
            if (!apart(r, u)) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: a result overlaps an upstream gradient");
        if (!apart(u, Extent{(uintptr_t)hd->ws_dev, 1, need, 0})) return fail(Q1ENV_ERR_INVALID_ARG, "q1env_head_backward: the workspace overlaps an upstream gradient");
    }
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

extern "C" {

int q1env_head_forward(int device, void* stream, const q1env_head* hd, int reduction, float* logp, float* entropy, float* loss) {
    return no_throw("q1env_head_forward", [&] { return head_forward(device, stream, hd, reduction, logp, entropy, loss); });
}

int q1env_head_backward(int device, void* stream, const q1env_head* hd, const float* dlogp, const float* dentropy, const float* dloss, void* dhidden, int64_t dhidden_stride,
                        void* dweight, int64_t dweight_stride, void* dbias) {
    return no_throw("q1env_head_backward", [&] { return head_backward(device, stream, hd, dlogp, dentropy, dloss, dhidden, dhidden_stride, dweight, dweight_stride, dbias); });
}

}  // extern "C"
