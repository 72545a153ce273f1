// q1env_clip.hip - the global norm of many gradient tensors and clipping by it (include/q1env.h q1env_grad_norm / q1env_grad_clip).
//
//   norm = |scale| sqrt(sum over all tensors of g^2);   out = g x scale x (norm <= max_norm ? 1 : max_norm / norm)
//
// Two passes: squares summed in float64 (no overflow or underflow of a float32 gradient's square, and an order fixed by the sizes alone: the
// same bits every time), one partial per workgroup; then every workgroup adds the partials up in the same order - cheaper than a third
// launch - and writes its share, last values first: those the device's last-level cache still holds from the first pass.  Up to SLOTS table slots travel in the kernel
// arguments; longer lists are first written to the workspace by small launches that carry SLOTS each.  Nothing is uploaded or kept between calls, and a captured
// launch holds its own table.
// Bound: memory.  536 870 913 float32 values (2.1 GB read, read again, written): 366 - 372 us for the first pass (5.8 TB/s), 795 - 807 for the second (5.4 TB/s; a plain copy makes 4.8).
#include "q1env_host.hpp"

#include <float.h>

#include <algorithm>

namespace {

constexpr int SLOTS = 120;                        // 32 bytes each: under 4 KB of kernel arguments
constexpr int THREADS = 256;
constexpr int MAX_BLOCKS = 2048, MAX_CLIP_BLOCKS = 1024;      // eight workgroups per CU for the pass that reads, four for the one that reads and writes (794 us against 909)
constexpr int64_t UNIT_MIN = 1024, UNIT_MAX = 8192;      // values a workgroup takes at a time

constexpr uint32_t PITCHED = 16, LAYOUT = 32;     // kinds of slot besides the dtype
struct Slot {
    const void* src;                              // LAYOUT (the slot behind a pitched tensor's): values per row
    void* dst;                                    // LAYOUT: values from row to row of src
    int64_t count;                                // LAYOUT: of dst
    uint32_t first;                               // first unit of the tensor
    uint32_t kind;
};
struct Table {
    Slot t[SLOTS];
    uint32_t n, units, unit, pad;
};
static_assert(sizeof(Table) <= 4000, "the table has to fit the kernel arguments");

template <int DT> struct El { typedef uint16_t type; };
template <> struct El<Q1ENV_DT_F32> { typedef float type; };
template <int DT> __device__ __forceinline__ float value(typename El<DT>::type v) {
    if constexpr (DT == Q1ENV_DT_F32) return v;
    else if constexpr (DT == Q1ENV_DT_BF16) return __builtin_bit_cast(float, (uint32_t)v << 16);
    else return (float)__builtin_bit_cast(_Float16, v);
}
template <int DT> __device__ __forceinline__ typename El<DT>::type rounded(float v) {
    if constexpr (DT == Q1ENV_DT_F32) return v;
    else if constexpr (DT == Q1ENV_DT_BF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
    else return __builtin_bit_cast(uint16_t, (_Float16)v);
}

__device__ __forceinline__ double block_sum(double a, double* red) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) a += __shfl_down(a, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

// runs f(slot, first value, end) over units blockIdx.x, blockIdx.x + gridDim.x, ... (neighbouring workgroups stream neighbouring memory), forwards or backwards
template <bool BACK, typename F> __device__ __forceinline__ void each_unit(const Slot* __restrict__ t, uint32_t n, uint32_t units, uint32_t unit, F f) {
    const uint32_t mine = blockIdx.x < units ? (units - 1 - blockIdx.x) / gridDim.x + 1 : 0;
    uint32_t lo = 0, hi = n;                      // where the slot is looked for
    for (uint32_t i = 0; i < mine; ++i) {
        const uint32_t u = blockIdx.x + (BACK ? mine - 1 - i : i) * gridDim.x;
        if (BACK) lo = 0;
        else hi = n;
        while (hi - lo > 1) {                     // the last slot whose first unit is <= u
            const uint32_t mid = (lo + hi) >> 1;
            if (t[mid].first <= u) lo = mid;
            else hi = mid;
        }
        const uint32_t at = t[lo].kind & LAYOUT ? lo - 1 : lo;
        const int64_t a = (int64_t)(u - t[at].first) * unit, count = t[at].count;
        f(t + at, a, a + unit < count ? a + unit : count);
    }
}

template <int DT> __device__ __forceinline__ double squares(const Slot* t, int64_t a, int64_t b, double acc) {
    typedef typename El<DT>::type E;
    constexpr int V = 16 / sizeof(E);
    const E* p = (const E*)t->src;
    if (t->kind & PITCHED) {
        const int64_t cols = (int64_t)t[1].src, pitch = (int64_t)t[1].dst;
        for (int64_t i = a + threadIdx.x; i < b; i += THREADS) {
            const int64_t r = i / cols;
            const double x = (double)value<DT>(p[r * pitch + (i - r * cols)]);
            acc = fma(x, x, acc);
        }
        return acc;
    }
    int64_t i = a + (int64_t)threadIdx.x * V;
    for (; i + V <= b; i += THREADS * V) {
        E v[V];
        __builtin_memcpy(v, p + i, 16);
#pragma unroll
        for (int j = 0; j < V; ++j) { const double x = (double)value<DT>(v[j]); acc = fma(x, x, acc); }
    }
    for (; i < b; ++i) { const double x = (double)value<DT>(p[i]); acc = fma(x, x, acc); }
    return acc;
}

// FAR: a factor outside float32's normal range (a norm or a scale beyond it) would lose its bits, or all of it: the product is a float64's
template <int DT, bool FAR> __device__ __forceinline__ void scaled(const Slot* t, int64_t a, int64_t b, double factor) {
    typedef typename El<DT>::type E;
    constexpr int V = 16 / sizeof(E);
    const E* p = (const E*)t->src;
    E* q = (E*)t->dst;
    const float c = (float)factor;
    auto times = [&](E x) { return rounded<DT>(FAR ? (float)((double)value<DT>(x) * factor) : value<DT>(x) * c); };
    if (!FAR && c == 1.0f && (const E*)q == p) return;                                   // in place and nothing to clip
    if (t->kind & PITCHED) {
        const int64_t cols = (int64_t)t[1].src, ps = (int64_t)t[1].dst, pd = t[1].count;
        for (int64_t i = a + threadIdx.x; i < b; i += THREADS) {
            const int64_t r = i / cols, k = i - r * cols;
            q[r * pd + k] = times(p[r * ps + k]);
        }
        return;
    }
    int64_t i = a + (int64_t)threadIdx.x * V;
    for (; i + V <= b; i += THREADS * V) {
        E w[V];
        __builtin_memcpy(w, p + i, 16);
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = times(w[j]);
        __builtin_memcpy(q + i, w, 16);
    }
    for (; i < b; ++i) q[i] = times(p[i]);
}

__device__ __forceinline__ void squares_of(const Slot* t, uint32_t n, uint32_t units, uint32_t unit, double* __restrict__ partial, double* red) {
    double acc = 0.0;
    each_unit<false>(t, n, units, unit, [&](const Slot* s, int64_t a, int64_t b) {
        const uint32_t dt = s->kind & 15;
        acc = dt == Q1ENV_DT_F32 ? squares<Q1ENV_DT_F32>(s, a, b, acc) : dt == Q1ENV_DT_BF16 ? squares<Q1ENV_DT_BF16>(s, a, b, acc) : squares<Q1ENV_DT_F16>(s, a, b, acc);
    });
    acc = block_sum(acc, red);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// the norm (before the scale) from the partials, the same in every workgroup
__device__ __forceinline__ double norm_of(const double* __restrict__ partial, int n, double* red) {
    double a = 0.0;
    for (int i = threadIdx.x; i < n; i += THREADS) a += partial[i];
    return sqrt(block_sum(a, red));
}

__global__ void __launch_bounds__(THREADS) norm_kernel(const double* __restrict__ partial, int n, double scale, float* __restrict__ norm) {
    __shared__ double red[4];
    const double v = norm_of(partial, n, red);
    if (threadIdx.x == 0) *norm = (float)(v * scale);
}

__device__ __forceinline__ void clip_of(const Slot* t, uint32_t n, uint32_t units, uint32_t unit, const double* __restrict__ partial, int parts, double scale, double max_norm,
                                        float* __restrict__ norm, double* red) {
    const double v = norm_of(partial, parts, red);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)(v * scale);
    const double c = v * scale <= max_norm ? scale : max_norm / v;               // a NaN norm makes every value NaN
    const bool far = c > 0.0 && (c < (double)FLT_MIN || c > (double)FLT_MAX);
    each_unit<true>(t, n, units, unit, [&](const Slot* s, int64_t a, int64_t b) {
        const uint32_t dt = s->kind & 15;
        if (far) {
            if (dt == Q1ENV_DT_F32) scaled<Q1ENV_DT_F32, true>(s, a, b, c);
            else if (dt == Q1ENV_DT_BF16) scaled<Q1ENV_DT_BF16, true>(s, a, b, c);
            else scaled<Q1ENV_DT_F16, true>(s, a, b, c);
        } else {
            if (dt == Q1ENV_DT_F32) scaled<Q1ENV_DT_F32, false>(s, a, b, c);
            else if (dt == Q1ENV_DT_BF16) scaled<Q1ENV_DT_BF16, false>(s, a, b, c);
            else scaled<Q1ENV_DT_F16, false>(s, a, b, c);
        }
    });
}

// the table in the kernel arguments, or in the workspace
__global__ void __launch_bounds__(THREADS) squares_kernel(Table tb, double* __restrict__ partial) {
    __shared__ double red[4];
    squares_of(tb.t, tb.n, tb.units, tb.unit, partial, red);
}
__global__ void __launch_bounds__(THREADS) squares_long_kernel(const Slot* __restrict__ t, uint32_t n, uint32_t units, uint32_t unit, double* __restrict__ partial) {
    __shared__ double red[4];
    squares_of(t, n, units, unit, partial, red);
}
__global__ void __launch_bounds__(THREADS) clip_kernel(Table tb, const double* __restrict__ partial, int parts, double scale, double max_norm, float* __restrict__ norm) {
    __shared__ double red[4];
    clip_of(tb.t, tb.n, tb.units, tb.unit, partial, parts, scale, max_norm, norm, red);
}
__global__ void __launch_bounds__(THREADS) clip_long_kernel(const Slot* __restrict__ t, uint32_t n, uint32_t units, uint32_t unit, const double* __restrict__ partial, int parts,
                                                            double scale, double max_norm, float* __restrict__ norm) {
    __shared__ double red[4];
    clip_of(t, n, units, unit, partial, parts, scale, max_norm, norm, red);
}
__global__ void __launch_bounds__(THREADS) table_kernel(Table tb, Slot* __restrict__ out) {
    for (uint32_t i = threadIdx.x; i < tb.n; i += THREADS) out[i] = tb.t[i];
}

size_t elem_size(int dt) { return dt == Q1ENV_DT_F32 ? 4 : 2; }

// what a call hands over, and how it is cut into launches
struct Job {
    int count;
    const void* const* src;
    void* const* dst;
    const int64_t* values;
    const int32_t* dtype;
    const int64_t *cols, *src_pitch, *dst_pitch;
};

struct Span { Extent x; int i; };
uintptr_t end_of(const Extent& x) { return x.at + (uintptr_t)(x.rows - 1) * x.pitch + x.row; }

// own: the norm and the workspace, which the call writes besides
int check_job(const char* who, const Job& j, bool write, const Extent (&own)[2]) {
    if (j.count < 0 || j.count > 65536) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": tensor count out of range (0 .. 65536)");
    if (j.count > 0 && (!j.src || !j.values || !j.dtype || (write && !j.dst))) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": null argument");
    if (j.cols && (!j.src_pitch || (write && !j.dst_pitch))) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": pitched tensors need their pitches");
    int64_t total = 0;
    for (int i = 0; i < j.count; ++i) {
        const int dt = j.dtype[i];
        if (dt != Q1ENV_DT_F32 && dt != Q1ENV_DT_BF16 && dt != Q1ENV_DT_F16) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": unknown dtype");
        if (j.values[i] < 0 || j.values[i] > (int64_t)1 << 40) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": a tensor's size is out of range");
        total += j.values[i];
        if (j.values[i] == 0) continue;
        if (!j.src[i] || (write && !j.dst[i])) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": a tensor's address is NULL");
        if ((uintptr_t)j.src[i] % elem_size(dt) || (write && (uintptr_t)j.dst[i] % elem_size(dt)))
            return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": an address is not aligned to its element size");
        if (j.cols && j.cols[i] != 0) {
            const int64_t c = j.cols[i];
            if (c < 0 || c > INT32_MAX || j.values[i] % c || j.src_pitch[i] < c || j.src_pitch[i] > INT32_MAX || (write && (j.dst_pitch[i] < c || j.dst_pitch[i] > INT32_MAX)))
                return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": bad columns / pitch of a pitched tensor");
        }
    }
    if (total > (int64_t)1 << 42) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": more than 2^42 values");
    bool free = apart(own[0], own[1]);
    for (int i = 0; i < j.count && free; ++i) {
        const uintptr_t es = elem_size(j.dtype[i]);
        const bool pitched = j.cols && j.cols[i] && j.values[i];
        const int64_t c = pitched ? j.cols[i] : j.values[i], rows = pitched ? j.values[i] / c : 1;
        for (const Extent& o : own)
            free = free && apart(o, Extent{(uintptr_t)j.src[i], rows, c * es, pitched ? (uintptr_t)j.src_pitch[i] * es : 0}) &&
                   (!write || apart(o, Extent{(uintptr_t)j.dst[i], rows, c * es, pitched ? (uintptr_t)j.dst_pitch[i] * es : 0}));
    }
    if (!free) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": the norm or the workspace overlaps a tensor or the other");
    if (!write) return 0;
    // no value is written by one tensor and read or written by another: every destination against all spans
    std::vector<Span> s;
    s.reserve(2 * (size_t)j.count);
    for (int i = 0; i < j.count; ++i) {
        if (j.values[i] == 0) continue;
        const uintptr_t es = elem_size(j.dtype[i]);
        const int64_t c = j.cols && j.cols[i] ? j.cols[i] : j.values[i], rows = j.values[i] / c;
        const uintptr_t sp = j.cols && j.cols[i] ? (uintptr_t)j.src_pitch[i] * es : 0, dp = j.cols && j.cols[i] ? (uintptr_t)j.dst_pitch[i] * es : 0;
        const uintptr_t sa = (uintptr_t)j.src[i], da = (uintptr_t)j.dst[i];
        s.push_back({{da, rows, c * es, dp}, i});
        if (sa != da || sp != dp) s.push_back({{sa, rows, c * es, sp}, ~i});      // ~i: a source
    }
    const auto before = [](const Span& x, const Span& y) { return x.x.at < y.x.at; };
    if (!std::is_sorted(s.begin(), s.end(), before)) std::sort(s.begin(), s.end(), before);
    std::vector<size_t> open;
    for (size_t k = 0; k < s.size(); ++k) {
        size_t kept = 0;
        for (size_t o : open) {
            if (end_of(s[o].x) <= s[k].x.at) continue;
            open[kept++] = o;
            if ((s[o].i >= 0 || s[k].i >= 0) && !apart(s[o].x, s[k].x))
                return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": a result overlaps another tensor (the same tensor twice, or a destination that is not its own source)");
        }
        open.resize(kept);
        open.push_back(k);
    }
    return 0;
}

int64_t unit_of(const Job& j) {
    int64_t total = 0;
    for (int i = 0; i < j.count; ++i) total += j.values[i];
    int64_t unit = UNIT_MIN;
    while (unit < UNIT_MAX && total / unit > MAX_BLOCKS) unit *= 2;
    return unit;
}

int run(const char* who, int device, hipStream_t stream, const Job& j, bool write, double scale, double max_norm, float* norm, void* ws, uint64_t ws_bytes) {
    const Extent own[2] = {{(uintptr_t)norm, 1, 4, 0}, {(uintptr_t)ws, 1, q1env_grad_norm_workspace_bytes(j.count), 0}};
    if (int rc = check_job(who, j, write, own)) return rc;
    if (!norm) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": norm is NULL");
    if (!(scale > 0.0) || std::isinf(scale)) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": scale must be positive and finite");
    if (write && !(max_norm >= 0.0)) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": max_norm must not be negative or NaN");
    if ((uintptr_t)ws % 8 || (uintptr_t)norm % 4) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": workspace / norm is not aligned (8 / 4 bytes)");
    if (!ws || ws_bytes < q1env_grad_norm_workspace_bytes(j.count)) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": workspace smaller than q1env_grad_norm_workspace_bytes");
    const int64_t unit = unit_of(j);
    for (int i = 0; i < j.count; ++i)
        if (j.values[i] / unit > (int64_t)1 << 30) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": a tensor's size is out of range");
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n == 0) return fail(Q1ENV_ERR_NO_DEVICE, std::string(who) + ": no HIP device (there is no CPU fallback)");
    if (device < 0 || device >= n) return fail(Q1ENV_ERR_INVALID_ARG, std::string(who) + ": no such device");
    DeviceGuard guard(device);
    double* partial = (double*)ws;
    // the slots, straight into the table that a launch takes
    Table tb;
    tb.n = 0;
    tb.unit = (uint32_t)unit;
    tb.pad = 0;
    Slot* const far = (Slot*)((char*)ws + 8 * MAX_BLOCKS);
    uint64_t units = 0;
    uint32_t slots = 0;                           // in the workspace already
    auto spill = [&]() -> int {
        hipLaunchKernelGGL(table_kernel, dim3(1), dim3(THREADS), 0, stream, tb, far + slots);
        HIP_TRY(hipGetLastError());
        slots += tb.n;
        tb.n = 0;
        return 0;
    };
    for (int i = 0; i < j.count; ++i) {
        if (j.values[i] == 0) continue;
        const bool pitched = j.cols && j.cols[i] != 0;
        if (tb.n + (pitched ? 2 : 1) > SLOTS)
            if (int rc = spill()) return rc;
        tb.t[tb.n++] = Slot{j.src[i], j.dst ? j.dst[i] : nullptr, j.values[i], (uint32_t)units, (uint32_t)j.dtype[i] | (pitched ? PITCHED : 0)};
        if (pitched) tb.t[tb.n++] = Slot{(const void*)j.cols[i], (void*)j.src_pitch[i], j.dst_pitch ? j.dst_pitch[i] : 0, (uint32_t)units, LAYOUT};
        units += (uint64_t)((j.values[i] + unit - 1) / unit);
    }
    const bool lng = slots > 0;
    if (lng && tb.n > 0)
        if (int rc = spill()) return rc;
    tb.units = (uint32_t)units;
    const unsigned blocks = (unsigned)std::min<uint64_t>(units, MAX_BLOCKS);
    if (blocks > 0) {
        if (lng) hipLaunchKernelGGL(squares_long_kernel, dim3(blocks), dim3(THREADS), 0, stream, far, slots, tb.units, tb.unit, partial);
        else hipLaunchKernelGGL(squares_kernel, dim3(blocks), dim3(THREADS), 0, stream, tb, partial);
        HIP_TRY(hipGetLastError());
    }
    const unsigned clip_blocks = std::min<unsigned>(blocks, MAX_CLIP_BLOCKS);
    if (!write || blocks == 0) hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(THREADS), 0, stream, partial, (int)blocks, scale, norm);
    else if (lng) hipLaunchKernelGGL(clip_long_kernel, dim3(clip_blocks), dim3(THREADS), 0, stream, far, slots, tb.units, tb.unit, partial, (int)blocks, scale, max_norm, norm);
    else hipLaunchKernelGGL(clip_kernel, dim3(clip_blocks), dim3(THREADS), 0, stream, tb, partial, (int)blocks, scale, max_norm, norm);
    HIP_TRY(hipGetLastError());
    return Q1ENV_OK;
}

}  // namespace

extern "C" {

uint64_t q1env_grad_norm_workspace_bytes(int count) {
    // a partial per workgroup, and a long list's table (two slots for a pitched tensor)
    return count < 0 || count > 65536 ? 0 : 8ull * MAX_BLOCKS + (2 * count > SLOTS ? 2 * sizeof(Slot) * (uint64_t)count : 0);
}

int q1env_grad_norm(int device, void* stream, int count, const void* const* src, const int64_t* values, const int32_t* dtype, const int64_t* cols, const int64_t* pitch, double scale,
                    float* norm, void* ws, uint64_t ws_bytes) {
    const Job j{count, src, nullptr, values, dtype, cols, pitch, nullptr};
    return no_throw("q1env_grad_norm", [&] { return run("q1env_grad_norm", device, (hipStream_t)stream, j, false, scale, 0.0, norm, ws, ws_bytes); });
}

int q1env_grad_clip(int device, void* stream, int count, const void* const* src, void* const* dst, const int64_t* values, const int32_t* dtype, const int64_t* cols,
                    const int64_t* src_pitch, const int64_t* dst_pitch, double scale, double max_norm, float* norm, void* ws, uint64_t ws_bytes) {
    const Job j{count, src, dst, values, dtype, cols, src_pitch, dst_pitch};
    return no_throw("q1env_grad_clip", [&] { return run("q1env_grad_clip", device, (hipStream_t)stream, j, true, scale, max_norm, norm, ws, ws_bytes); });
}

}  // extern "C"
