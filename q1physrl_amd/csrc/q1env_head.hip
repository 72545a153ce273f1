// q1env_head.hip - the wide categorical head of libq1env.so (include/q1env.h q1env_head_*): log-probability, entropy and cross entropy of given
// classes from hidden rows and the head's weights without the logits ever being kept, and the gradients (kernels: q1head.hpp).
#include "q1env_host.hpp"
#include "q1head.hpp"

using namespace q1head;

namespace {

constexpr uint64_t PIECE_BYTES = 256ull << 20;     // of the gradient of one piece of the classes
constexpr int64_t MAX_ROWS = 1 << 22, MAX_WIDTH = 1 << 16, MAX_CLASSES = 1 << 22;
constexpr int64_t WORKGROUPS = 512;                // two per CU: what a launch should have before its sums are split further

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
uint64_t aligned(uint64_t x) { return (x + 255) & ~255ull; }
size_t elem_size(int dt) { return dt == F32 ? 4 : 2; }

// the forward pass's results as the backward pass reads them (q1env_head_state_bytes)
struct State {
    float *lse, *entropy, *each;
    int64_t* target;
    uint8_t* live;
    static uint64_t bytes(int64_t n) { return 2 * aligned(4 * n) + aligned(8 * n) + aligned(n) + 256; }
    State(void* p, int64_t n) {
        char* c = (char*)p;
        lse = (float*)c; c += aligned(4 * n);
        entropy = (float*)c; c += aligned(4 * n);
        target = (int64_t*)c; c += aligned(8 * n);
        live = (uint8_t*)c; c += aligned(n);
        each = (float*)c;
    }
};

struct Plan {
    int64_t piece, pieces;             // classes per piece (a multiple of BM)
    int dh_split, dw_split;
    int64_t dh_k, dw_k;                // classes / rows per split
    uint64_t part, own, scale, g, db, dh_slab, dw_slab;        // byte offsets in the workspace
    uint64_t forward_bytes, backward_bytes;
};

void split(int64_t tiles, int64_t k, int& n, int64_t& len) {
    int64_t s = div_up(WORKGROUPS, tiles), most = div_up(k, 512);        // a part shorter than 512 costs more in its slab than it gains
    if (s > most) s = most;
    if (s < 1) s = 1;
    len = div_up(div_up(k, s), BK) * BK;
    n = (int)div_up(k, len);
}

Plan plan_of(int dt, int64_t rows, int64_t width, int64_t classes) {
    Plan p{};
    const int64_t ct = div_up(classes, BM);
    p.own = 0;
    p.part = aligned(4 * rows);
    p.forward_bytes = p.part + aligned(12 * (uint64_t)ct * rows);
    int64_t piece = (int64_t)(PIECE_BYTES / (elem_size(dt) * rows)) / BM * BM;
    if (piece < BM) piece = BM;
    if (piece > ct * BM) piece = ct * BM;
    p.piece = piece;
    p.pieces = div_up(classes, piece);
    split(div_up(width, BM) * div_up(rows, BN), piece, p.dh_split, p.dh_k);
    split(div_up(width, BM) * div_up(piece, BN), rows, p.dw_split, p.dw_k);
    uint64_t at = 0;
    p.scale = at; at += 256;
    p.g = at; at += aligned(elem_size(dt) * (uint64_t)rows * piece);
    p.db = at; at += aligned(4 * (uint64_t)div_up(rows, BN) * classes);
    p.dh_slab = at;
    if (p.dh_split > 1 || p.pieces > 1) at += aligned(4 * (uint64_t)p.dh_split * rows * width);
    p.dw_slab = at;
    if (p.dw_split > 1) at += aligned(4 * (uint64_t)p.dw_split * piece * width);
    p.backward_bytes = at;
    return p;
}

Operand operand(int dt, const void* p, int64_t stride, int64_t extent, const uint8_t* live = nullptr) {
    const bool vec = ((uintptr_t)p & 15) == 0 && (stride * (int64_t)elem_size(dt)) % 16 == 0;
    return Operand{p, stride, extent, live, vec ? 1 : 0};
}

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

template <int DT>
int forward(hipStream_t stream, const q1env_head& q, const Plan& p, int reduction, float* logp, float* entropy, float* loss) {
    const int64_t n = q.rows;
    State st(q.state_dev, n);
    char* ws = (char*)q.ws_dev;
    const dim3 rows256((unsigned)div_up(n, 256));
    if (n > 0) {
        if (q.target_bits == 64)
            hipLaunchKernelGGL((prepare_kernel<int64_t>), rows256, dim3(256), 0, stream, (const int64_t*)q.target_dev, n, q.classes, q.ignore_index, st.target, st.live);
        else
            hipLaunchKernelGGL((prepare_kernel<int32_t>), rows256, dim3(256), 0, stream, (const int32_t*)q.target_dev, n, q.classes, q.ignore_index, st.target, st.live);
        HIP_TRY(hipGetLastError());
        const Head hd{operand(DT, q.weight_dev, q.weight_stride, q.classes), operand(DT, q.hidden_dev, q.hidden_stride, n), q.bias_dev, st.target, n, q.width, q.classes};
        const int64_t tiles = div_up(q.classes, BM);
        hipLaunchKernelGGL((statistics_kernel<DT>), dim3((unsigned)tiles, (unsigned)div_up(n, BN)), dim3(256), 0, stream, hd, (float*)(ws + p.part), (float*)(ws + p.own));
        HIP_TRY(hipGetLastError());
        hipLaunchKernelGGL(join_kernel, dim3((unsigned)div_up(n, 16)), dim3(256), 0, stream, (const float*)(ws + p.part), (const float*)(ws + p.own), st.target, n, (int)tiles,
                           logp, entropy, st.entropy, st.lse);
        HIP_TRY(hipGetLastError());
    }
    if (loss) {
        hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(1024), 0, stream, logp, st.live, n, reduction == Q1ENV_REDUCE_MEAN ? 1 : 0, loss, st.each);
        HIP_TRY(hipGetLastError());
    }
    return Q1ENV_OK;
}

template <int DT>
int backward(hipStream_t stream, const q1env_head& q, const Plan& p, Upstream up, void* dh, int64_t dh_stride, void* dw, int64_t dw_stride, void* db) {
    const int64_t n = q.rows, v = q.classes, d = q.width;
    State st(q.state_dev, n);
    char* ws = (char*)q.ws_dev;
    float* scale = (float*)(ws + p.scale);
    up.scale = scale;
    up.each = up.dloss ? st.each : nullptr;
    hipLaunchKernelGGL(scale_kernel, dim3(1), dim3(1024), 0, stream, up, st.live, n, DT == F16 ? 1 : 0, scale);
    HIP_TRY(hipGetLastError());
    const Head hd{operand(DT, q.weight_dev, q.weight_stride, v), operand(DT, q.hidden_dev, q.hidden_stride, n), q.bias_dev, st.target, n, d, v};
    const unsigned row_tiles = (unsigned)div_up(n, BN), width_tiles = (unsigned)div_up(d, BM);
    void* g = ws + p.g;
    float *dh_slab = p.dh_split > 1 || p.pieces > 1 ? (float*)(ws + p.dh_slab) : nullptr, *dw_slab = p.dw_split > 1 ? (float*)(ws + p.dw_slab) : nullptr;
    const size_t es = elem_size(DT);
    for (int64_t c0 = 0; c0 < v; c0 += p.piece) {
        const int64_t c1 = c0 + p.piece < v ? c0 + p.piece : v, len = c1 - c0;
        hipLaunchKernelGGL((gradient_kernel<DT>), dim3((unsigned)div_up(len, BM), row_tiles), dim3(256), 0, stream, hd, up, c0, c1, p.piece, st.lse, st.entropy, g,
                           db ? (float*)(ws + p.db) : nullptr);
        HIP_TRY(hipGetLastError());
        if (dw) {
            Product pr{operand(DT, q.hidden_dev, q.hidden_stride, d, st.live), operand(DT, g, p.piece, len), n, p.dw_k, len, d, (char*)dw + es * c0 * dw_stride, dw_stride,
                       dw_slab, 0, scale, nullptr};
            hipLaunchKernelGGL((product_kernel<DT, true, true>), dim3(width_tiles, (unsigned)div_up(len, BN), (unsigned)p.dw_split), dim3(256), 0, stream, pr);
            HIP_TRY(hipGetLastError());
            if (dw_slab) {
                hipLaunchKernelGGL((finish_kernel<DT>), dim3((unsigned)div_up(len * d, 256)), dim3(256), 0, stream, dw_slab, p.dw_split, len, d, scale, (const uint8_t*)nullptr, pr.out,
                                   dw_stride);
                HIP_TRY(hipGetLastError());
            }
        }
        if (dh) {
            Product pr{operand(DT, (const char*)q.weight_dev + es * c0 * q.weight_stride, q.weight_stride, d), operand(DT, g, p.piece, n), len, p.dh_k, n, d, dh, dh_stride,
                       dh_slab, c0 > 0 ? 1 : 0, scale, st.live};
            hipLaunchKernelGGL((product_kernel<DT, true, false>), dim3(width_tiles, row_tiles, (unsigned)p.dh_split), dim3(256), 0, stream, pr);
            HIP_TRY(hipGetLastError());
        }
    }
    if (dh && dh_slab) {
        hipLaunchKernelGGL((finish_kernel<DT>), dim3((unsigned)div_up(n * d, 256)), dim3(256), 0, stream, dh_slab, p.dh_split, n, d, scale, st.live, dh, dh_stride);
        HIP_TRY(hipGetLastError());
    }
    if (db) {
        hipLaunchKernelGGL((bias_kernel<DT>), dim3((unsigned)div_up(v, 256)), dim3(256), 0, stream, (const float*)(ws + p.db), v, (int)row_tiles, scale, db);
        HIP_TRY(hipGetLastError());
    }
    return Q1ENV_OK;
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
    const Plan p = plan_of(dtype, rows, width, classes);
    return backward ? p.backward_bytes : p.forward_bytes;
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
    const Plan p = hd->rows > 0 ? plan_of(hd->dtype, hd->rows, hd->width, hd->classes) : Plan{};
    switch (hd->dtype) {
        case Q1ENV_DT_F32: return forward<F32>((hipStream_t)stream, *hd, p, reduction, logp, entropy, loss);
        case Q1ENV_DT_BF16: return forward<BF16>((hipStream_t)stream, *hd, p, reduction, logp, entropy, loss);
        default: return forward<F16>((hipStream_t)stream, *hd, p, reduction, logp, entropy, loss);
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
    const Plan p = plan_of(hd->dtype, hd->rows, hd->width, hd->classes);
    const Upstream up{dlogp, dentropy, dloss, nullptr, nullptr};
    switch (hd->dtype) {
        case Q1ENV_DT_F32: return backward<F32>((hipStream_t)stream, *hd, p, up, dhidden, dhidden_stride, dweight, dweight_stride, dbias);
        case Q1ENV_DT_BF16: return backward<BF16>((hipStream_t)stream, *hd, p, up, dhidden, dhidden_stride, dweight, dweight_stride, dbias);
        default: return backward<F16>((hipStream_t)stream, *hd, p, up, dhidden, dhidden_stride, dweight, dweight_stride, dbias);
    }
}

}  // extern "C"
