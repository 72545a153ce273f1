// q1head.hpp - device code of the wide categorical head (q1env_head.hip): softmax statistics of logits that are never stored, and the three
// products of their gradient, as tiled matrix-core kernels.
//
//   l_ij = h_i . w_j + b_j            i: sample (row of hidden), j: class (row of weight)
//   lse_i = log sum_j exp l_ij,  logp_i = l_i,t(i) - lse_i,  H_i = lse_i - sum_j p_ij l_ij
//   g_ij = A_i ([j = t_i] - p_ij) - E_i p_ij (log p_ij + H_i)        for upstream A_i = d/dlogp_i, E_i = d/dH_i
//   dh = g W,  dW = g^T h,  db = sum_i g_i
//
// Operand precision: float16 / bfloat16 inputs feed v_mfma_f32_32x32x16 as they are.  A float32 value travels as THREE bfloat16 pieces
// a = a1 + a2 + a3 (8 + 8 + 8 significant bits: exact) and a product is the six largest of the nine piece products, a1 b1, a1 b2, a2 b1, a1 b3,
// a3 b1, a2 b2; what is dropped is below 2^-26 of |a b|, under the rounding of the float32 accumulator the products go to.  (The float32
// matrix instruction runs at 1/16 of the bfloat16 one; six products run at 1/6.)
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace q1head {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;

constexpr int F32 = 0, BF16 = 1, F16 = 2;

template <int DT> struct Elem;
template <> struct Elem<F32> { typedef float type; static constexpr int planes = 3; };
template <> struct Elem<BF16> { typedef uint16_t type; static constexpr int planes = 1; };
template <> struct Elem<F16> { typedef uint16_t type; static constexpr int planes = 1; };

__device__ __forceinline__ uint16_t bf16_bits(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ float bf16_value(uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }
__device__ __forceinline__ uint16_t f16_bits(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
__device__ __forceinline__ float f16_value(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }

template <int DT> __device__ __forceinline__ float to_float(typename Elem<DT>::type v) {
    if constexpr (DT == F32) return v;
    else if constexpr (DT == BF16) return bf16_value(v);
    else return f16_value(v);
}
template <int DT> __device__ __forceinline__ typename Elem<DT>::type from_float(float v) {
    if constexpr (DT == F32) return v;
    else if constexpr (DT == BF16) return bf16_bits(v);
    else return f16_bits(v);
}

template <int DT> __device__ __forceinline__ f32x16 mfma(const u32x4& a, const u32x4& b, const f32x16& c) {
    if constexpr (DT == F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// exp(x) for x <= 0 (and -inf, NaN): one hardware exponential, with the rounding error of x log2(e) put back where the result is held in full
// precision (|x| 2^-24 relative otherwise)
__device__ __forceinline__ float exp_neg(float x) {
    const float t = x * 1.4426950408889634f;
    const float e = __builtin_amdgcn_exp2f(t);
    const float r = fmaf(x, 1.4426950408889634f, -t) + x * 1.925963033500e-8f;      // log2(e) - float32(log2(e))
    return t > -150.0f ? fmaf(e, r * 0.6931471805599453f, e) : e;
}

// ------------------------------------------------------------------------------------------------------------------------------
// C[m][n] = sum_k A(m, k) B(n, k), a BM x BN tile per workgroup of 256 lanes (2 x 2 waves of 64 x 64).
// An operand is (pointer, stride): K-major false: element (x, k) at p[x * stride + k] (k contiguous); true: p[k * stride + x].
struct Operand {
    const void* p;
    int64_t stride;             // elements
    int64_t extent;             // number of valid x
    const uint8_t* live;        // K-major only: where set, element (x, k) counts as zero when live[k] == 0 (whatever memory holds there)
    int vec;                    // 16-byte loads are aligned (pointer and stride)
};

constexpr int BM = 128, BN = 128, BK = 32, LDS_ROW = BK + 8;      // 80-byte rows: 16-byte aligned, and eight rows cover all 64 banks

template <int DT> struct Stage {                                    // one operand tile, [plane][x][k]
    uint16_t v[Elem<DT>::planes][BM][LDS_ROW];
};

template <int DT, bool KMAJOR> struct Loader {
    typedef typename Elem<DT>::type E;
    static constexpr int V = 16 / sizeof(E);                        // elements of a 16-byte load
    static constexpr int CHUNKS = BM * BK / V / 256;                // per lane
    E r[CHUNKS][V];

    // tile at (x0, k0); k < k_end
    __device__ __forceinline__ void load(const Operand& o, int64_t x0, int64_t k0, int64_t k_end) {
        const E* p = (const E*)o.p;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int i = c * 256 + (int)threadIdx.x;
            int64_t x, k;
            if constexpr (KMAJOR) { x = x0 + (i % (BM / V)) * V; k = k0 + i / (BM / V); }
            else { x = x0 + i / (BK / V); k = k0 + (i % (BK / V)) * V; }
            const bool row_ok = KMAJOR ? (k < k_end && (!o.live || o.live[k] != 0)) : x < o.extent;
            const int64_t left = row_ok ? (KMAJOR ? o.extent - x : k_end - k) : 0;      // valid elements from here on
            const E* q = KMAJOR ? p + k * o.stride + x : p + x * o.stride + k;
            if (left >= V && o.vec) {
                const u32x4 w = *(const u32x4*)q;
                __builtin_memcpy(r[c], &w, 16);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) r[c][j] = j < left ? q[j] : (E)0;
            }
        }
    }
    __device__ __forceinline__ void store(Stage<DT>& s) const {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int i = c * 256 + (int)threadIdx.x;
            const int x = KMAJOR ? (i % (BM / V)) * V : i / (BK / V), k = KMAJOR ? i / (BM / V) : (i % (BK / V)) * V;
            uint16_t piece[Elem<DT>::planes][V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if constexpr (DT == F32) {
                    const float a = r[c][j];
                    const uint16_t p1 = bf16_bits(a);
                    const float r1 = a - bf16_value(p1);
                    const uint16_t p2 = bf16_bits(r1);
                    piece[0][j] = p1; piece[1][j] = p2; piece[2][j] = bf16_bits(r1 - bf16_value(p2));
                } else
                    piece[0][j] = r[c][j];
            }
#pragma unroll
            for (int q = 0; q < Elem<DT>::planes; ++q) {
                if constexpr (KMAJOR) {
#pragma unroll
                    for (int j = 0; j < V; ++j) s.v[q][x + j][k] = piece[q][j];
                } else
                    __builtin_memcpy(&s.v[q][x][k], piece[q], 2 * V);
            }
        }
    }
};

// accumulator layout of v_mfma_f32_32x32x16: lane l holds column n = l % 32, register r holds row m = 8 (r / 4) + 4 (l / 32) + r % 4
struct Acc { f32x16 t[2][2]; };                                     // [m tile][n tile] of this wave's 64 x 64

template <int DT, bool AK, bool BK_>
__device__ __forceinline__ void gemm_tile(const Operand& a, const Operand& b, int64_t m0, int64_t n0, int64_t k_begin, int64_t k_end, Acc& acc,
                                          Stage<DT>& sa, Stage<DT>& sb) {
    constexpr int P = Elem<DT>::planes;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc.t[i][j][r] = 0.0f;
    Loader<DT, AK> la;
    Loader<DT, BK_> lb;
    la.load(a, m0, k_begin, k_end);
    lb.load(b, n0, k_begin, k_end);
    for (int64_t k = k_begin; k < k_end; k += BK) {
        __syncthreads();                                            // the previous tile has been read
        la.store(sa);
        lb.store(sb);
        __syncthreads();
        if (k + BK < k_end) {
            la.load(a, m0, k + BK, k_end);
            lb.load(b, n0, k + BK, k_end);
        }
#pragma unroll
        for (int kk = 0; kk < BK; kk += 16) {
            u32x4 fa[P][2], fb[P][2];
#pragma unroll
            for (int q = 0; q < P; ++q)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    fa[q][i] = *(const u32x4*)&sa.v[q][wm + 32 * i + (lane & 31)][kk + 8 * (lane >> 5)];
                    fb[q][i] = *(const u32x4*)&sb.v[q][wn + 32 * i + (lane & 31)][kk + 8 * (lane >> 5)];
                }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if constexpr (P == 3) {                         // smallest products first
                        acc.t[i][j] = mfma<DT>(fa[1][i], fb[1][j], acc.t[i][j]);
                        acc.t[i][j] = mfma<DT>(fa[0][i], fb[2][j], acc.t[i][j]);
                        acc.t[i][j] = mfma<DT>(fa[2][i], fb[0][j], acc.t[i][j]);
                        acc.t[i][j] = mfma<DT>(fa[0][i], fb[1][j], acc.t[i][j]);
                        acc.t[i][j] = mfma<DT>(fa[1][i], fb[0][j], acc.t[i][j]);
                    }
                    acc.t[i][j] = mfma<DT>(fa[0][i], fb[0][j], acc.t[i][j]);
                }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------------------
// what a launch over logit tiles knows of the head
struct Head {
    Operand w, h;                    // A: weight (m = class), B: hidden (n = row)
    const void* bias;
    const int64_t* target;           // classes as the prepare kernel wrote them: -1 = ignored, -2 = out of range
    int64_t rows, width, classes;
};

// classes widened to int64 with the two special values, and the liveness bytes
template <typename T>
__global__ void __launch_bounds__(256) prepare_kernel(const T* __restrict__ target, int64_t rows, int64_t classes, int64_t ignore, int64_t* __restrict__ out,
                                                      uint8_t* __restrict__ live) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows) return;
    const int64_t t = (int64_t)target[i];
    const bool ign = t == ignore;
    out[i] = ign ? -1 : (t < 0 || t >= classes ? -2 : t);
    live[i] = ign ? 0 : 1;
}

// statistics of a set of classes: maximum m, s = sum exp(l - m), u = sum (l - m) exp(l - m)
struct Stat { float m, s, u; };
__device__ __forceinline__ Stat joined(const Stat& a, const Stat& b) {
    const float m = fmaxf(a.m, b.m);
    // a set of classes at -inf has m = -inf, s = u = 0 and counts nothing; a difference is kept where 0 x (difference x s) is still 0 (masks of the type's lowest value)
    const float da = a.m == -INFINITY ? 0.0f : fmaxf(a.m - m, -1.0e30f), db = b.m == -INFINITY ? 0.0f : fmaxf(b.m - m, -1.0e30f);
    const float fa = a.m == -INFINITY ? 0.0f : exp_neg(da), fb = b.m == -INFINITY ? 0.0f : exp_neg(db);
    return Stat{m, fa * a.s + fb * b.s, fa * (a.u + da * a.s) + fb * (b.u + db * b.s)};
}

// class-tile statistics of each row: max m, s = sum exp(l - m), u = sum (l - m) exp(l - m); and the logit of the row's own class
template <int DT>
__global__ void __launch_bounds__(256) statistics_kernel(Head hd, float* __restrict__ part, float* __restrict__ own_logit) {
    __shared__ Stage<DT> sa, sb;
    __shared__ float red[2][BN][3];
    typedef typename Elem<DT>::type E;
    const int64_t m0 = (int64_t)blockIdx.x * BM, n0 = (int64_t)blockIdx.y * BN;
    Acc acc;
    gemm_tile<DT, false, false>(hd.w, hd.h, m0, n0, 0, hd.width, acc, sa, sb);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    const E* bias = (const E*)hd.bias;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int nl = wn + 32 * j + (lane & 31);
        const int64_t n = n0 + nl;
        const int64_t t = n < hd.rows ? hd.target[n] : -1;
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t m = m0 + wm + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                float l = acc.t[i][j][r];
                if (m < hd.classes) {
                    if (bias) l += to_float<DT>(bias[m]);
                    if (m == t) own_logit[n] = l;
                } else
                    l = -INFINITY;
                acc.t[i][j][r] = l;
                mx = fmaxf(mx, l);
            }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float s = 0.0f, u = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float d = acc.t[i][j][r] - ref, e = exp_neg(d);
                s += e;
                u = fmaf(fmaxf(d, -3.0e38f), e, u);                 // a class at -inf adds 0, not 0 x inf
            }
        s += __shfl_xor(s, 32, 64);
        u += __shfl_xor(u, 32, 64);
        if (lane < 32) { red[wave & 1][nl][0] = mx; red[wave & 1][nl][1] = s; red[wave & 1][nl][2] = u; }
    }
    __syncthreads();
    if (threadIdx.x < BN && n0 + threadIdx.x < hd.rows) {
        const int nl = threadIdx.x;
        const Stat t = joined(Stat{red[0][nl][0], red[0][nl][1], red[0][nl][2]}, Stat{red[1][nl][0], red[1][nl][1], red[1][nl][2]});
        float* o = part + 3 * (size_t)blockIdx.x * hd.rows + n0 + nl;
        o[0] = t.m; o[hd.rows] = t.s; o[2 * hd.rows] = t.u;
    }
}

// joins the tiles' statistics: 16 lanes per row, 16 rows per workgroup
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ part, const float* __restrict__ own_logit, const int64_t* __restrict__ target,
                                                   int64_t rows, int tiles, float* __restrict__ logp, float* __restrict__ entropy, float* __restrict__ entropy_kept,
                                                   float* __restrict__ lse) {
    __shared__ float red[3][16][17];
    const int r = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int64_t n = (int64_t)blockIdx.x * 16 + r;
    Stat a{-INFINITY, 0.0f, 0.0f};
    if (n < rows)
        for (int t = g; t < tiles; t += 16) {
            const float* o = part + 3 * (size_t)t * rows + n;
            a = joined(a, Stat{o[0], o[rows], o[2 * rows]});
        }
    red[0][g][r] = a.m; red[1][g][r] = a.s; red[2][g][r] = a.u;
    __syncthreads();
    if (threadIdx.x < 16 && n < rows) {
        for (int k = 1; k < 16; ++k) a = joined(a, Stat{red[0][k][r], red[1][k][r], red[2][k][r]});
        const int64_t t = target[n];
        const float ls = logf(a.s);
        float z = a.m + ls, h = ls - a.u / a.s, lp = 0.0f;
        if (t >= 0) lp = (own_logit[n] - a.m) - ls;
        else if (t == -1) { h = 0.0f; z = 0.0f; }                  // ignored
        else { lp = h = z = NAN; }                                  // a class that does not exist
        logp[n] = lp;
        if (entropy) entropy[n] = h;
        entropy_kept[n] = h;
        lse[n] = z;
    }
}

// loss[0] = -sum logp / max(1, live rows) or -sum logp; loss[1] = what d loss / d(-logp) of a live row is
__global__ void __launch_bounds__(1024) loss_kernel(const float* __restrict__ logp, const uint8_t* __restrict__ live, int64_t rows, int mean, float* __restrict__ loss,
                                                    float* __restrict__ each) {
    __shared__ double red[16];
    __shared__ int64_t cnt[16];
    double a = 0.0;
    int64_t c = 0;
    for (int64_t i = threadIdx.x; i < rows; i += 1024) { a += (double)logp[i]; c += live[i]; }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) { a += __shfl_down(a, off, 64); c += __shfl_down((long long)c, off, 64); }
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = a; cnt[threadIdx.x >> 6] = c; }
    __syncthreads();
    if (threadIdx.x == 0) {
        a = 0.0; c = 0;
        for (int k = 0; k < 16; ++k) { a += red[k]; c += cnt[k]; }
        const double n = mean ? (double)(c > 0 ? c : 1) : 1.0;
        loss[0] = (float)(0.0 - a / n);
        each[0] = (float)(1.0 / n);
    }
}

// ------------------------------------------------------------------------------------------------------------------------------
// The gradient's scale.  g is stored as it is in float32 and bfloat16.  Float16 loses what lies below 2^-24, so there the stored values are
// g / scale with a power of two `scale` that brings the largest possible |g| to 2^14, and the products' results are multiplied by it.
struct Upstream {
    const float* dlogp;              // per row, or null
    const float* dentropy;           // per row, or null
    const float* dloss;              // one value (with each): A_i = -dloss each for every live row
    const float* each;
    const float* scale;              // written by scale_kernel
};

// scale[0]: what stored values are multiplied by, scale[1]: what results are multiplied by
__global__ void __launch_bounds__(1024) scale_kernel(Upstream up, const uint8_t* __restrict__ live, int64_t rows, int f16, float* __restrict__ scale) {
    __shared__ float red[16];
    if (up.dloss) {                  // one factor for all rows: the stored values are p - [j = t], which need no further scale but float16's
        if (threadIdx.x == 0) { scale[0] = f16 ? 16384.0f : 1.0f; scale[1] = *up.dloss * *up.each * (f16 ? 0x1p-14f : 1.0f); }
        return;
    }
    if (!f16) {
        if (threadIdx.x == 0) { scale[0] = 1.0f; scale[1] = 1.0f; }
        return;
    }
    float mx = 0.0f;
    for (int64_t i = threadIdx.x; i < rows; i += 1024)
        if (live[i]) mx = fmaxf(mx, (up.dlogp ? fabsf(up.dlogp[i]) : 0.0f) + (up.dentropy ? 16.0f * fabsf(up.dentropy[i]) : 0.0f));   // |p (log p + H)| < 16 up to 2^22 classes
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_down(mx, off, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < 16; ++k) mx = fmaxf(mx, red[k]);
        int e = 0;
        if (mx > 0.0f && mx < INFINITY) (void)frexpf(mx, &e);       // mx in [2^(e-1), 2^e)
        e = e < -110 ? -110 : (e > 126 ? 126 : e);
        scale[0] = ldexpf(1.0f, 14 - e);
        scale[1] = ldexpf(1.0f, e - 14);
    }
}

// a piece [c0, c0 + piece) of the classes: the logits again, and the gradient of each -> g[row][class - c0] (stride `piece`), and the sums over
// this tile's rows -> db_part[row tile][class]
template <int DT>
__global__ void __launch_bounds__(256) gradient_kernel(Head hd, Upstream up, int64_t c0, int64_t c1, int64_t piece, const float* __restrict__ lse, const float* __restrict__ entropy,
                                                       void* __restrict__ g_out, float* __restrict__ db_part) {
    __shared__ Stage<DT> sa, sb;
    typedef typename Elem<DT>::type E;
    const int64_t m0 = c0 + (int64_t)blockIdx.x * BM, n0 = (int64_t)blockIdx.y * BN;
    Acc acc;
    gemm_tile<DT, false, false>(hd.w, hd.h, m0, n0, 0, hd.width, acc, sa, sb);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    const E* bias = (const E*)hd.bias;
    E* g = (E*)g_out;
    const float sc = up.scale[0];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t n = n0 + wn + 32 * j + (lane & 31);
        const int64_t t = n < hd.rows ? hd.target[n] : -1;
        const bool on = t != -1;
        const float z = on ? lse[n] : 0.0f, hrow = on && up.dentropy ? entropy[n] : 0.0f;
        const float A = on ? (up.dloss ? -1.0f : (up.dlogp ? up.dlogp[n] : 0.0f)) * sc : 0.0f, Ee = on && up.dentropy ? up.dentropy[n] * sc : 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int64_t m = m0 + wm + 32 * i + 8 * r4 + 4 * (lane >> 5);
                E q[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = 0.0f;
                    if (on && m + r < c1) {
                        float l = acc.t[i][j][4 * r4 + r];
                        if (bias) l += to_float<DT>(bias[m + r]);
                        const float d = l - z, p = exp_neg(d);
                        v = -A * p;
                        if (up.dentropy) v -= Ee * p * (fmaxf(d, -3.0e38f) + hrow);
                        if (m + r == t) v += A;
                    }
                    acc.t[i][j][4 * r4 + r] = v;
                    q[r] = from_float<DT>(v);
                }
                if (n < hd.rows && m < c0 + piece) __builtin_memcpy(g + n * piece + (m - c0), q, sizeof q);      // piece is a multiple of BM
            }
    }
    if (db_part) {
        float (*red)[BM] = (float (*)[BM])&sa;                       // [4][BM]: 2 column halves x 2 lane halves never write the same word
        __syncthreads();
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float v = acc.t[i][0][r] + acc.t[i][1][r];
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
                if ((lane & 31) == 0) red[wave >> 1][wm + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)] = v;
            }
        __syncthreads();
        if (threadIdx.x < BM && m0 + threadIdx.x < c1) db_part[(size_t)blockIdx.y * hd.classes + m0 + threadIdx.x] = red[0][threadIdx.x] + red[1][threadIdx.x];
    }
}

// db[class] = scale x sum over row tiles, in the order of the tiles
template <int DT>
__global__ void __launch_bounds__(256) bias_kernel(const float* __restrict__ part, int64_t classes, int tiles, const float* __restrict__ scale, void* __restrict__ out) {
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (j >= classes) return;
    float a = 0.0f;
    for (int t = 0; t < tiles; ++t) a += part[(size_t)t * classes + j];
    ((typename Elem<DT>::type*)out)[j] = from_float<DT>(a * scale[1]);
}

// out[n][m] (stride out_stride): m = column of the result (width), n = its row.  slab: the sums stay in float32 [split][rows][width] for
// finish_kernel (accumulate: added to what is there); without it the scaled result is stored.
struct Product {
    Operand a, b;
    int64_t k, split_k;                // length of the sum; part per z-slice (a multiple of BK)
    int64_t rows, width;               // of the result
    void* out;
    int64_t out_stride;
    float* slab;
    int accumulate;
    const float* scale;
    const uint8_t* live;               // result rows that are zero whatever the operands hold
};

template <int DT, bool AK, bool BK_>
__global__ void __launch_bounds__(256) product_kernel(Product pr) {
    __shared__ Stage<DT> sa, sb;
    const int64_t m0 = (int64_t)blockIdx.x * BM, n0 = (int64_t)blockIdx.y * BN;
    const int64_t kb = (int64_t)blockIdx.z * pr.split_k, ke = kb + pr.split_k < pr.k ? kb + pr.split_k : pr.k;
    Acc acc;
    gemm_tile<DT, AK, BK_>(pr.a, pr.b, m0, n0, kb, ke, acc, sa, sb);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    typedef typename Elem<DT>::type E;
    const float sc = pr.slab ? 1.0f : pr.scale[1];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t n = n0 + wn + 32 * j + (lane & 31);
        if (n >= pr.rows) continue;
        const bool on = !pr.live || pr.live[n];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t m = m0 + wm + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                if (m >= pr.width) continue;
                if (pr.slab) {
                    float* o = pr.slab + ((size_t)blockIdx.z * pr.rows + n) * pr.width + m;
                    *o = pr.accumulate ? *o + acc.t[i][j][r] : acc.t[i][j][r];
                } else
                    ((E*)pr.out)[n * pr.out_stride + m] = from_float<DT>(on ? acc.t[i][j][r] * sc : 0.0f);
            }
    }
}

// result = scale x sum of the slabs, in their order
template <int DT>
__global__ void __launch_bounds__(256) finish_kernel(const float* __restrict__ slab, int splits, int64_t rows, int64_t width, const float* __restrict__ scale,
                                                     const uint8_t* __restrict__ live, void* __restrict__ out, int64_t out_stride) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * width) return;
    const int64_t n = i / width, m = i - n * width;
    float a = 0.0f;
    if (!live || live[n]) {
        for (int s = 0; s < splits; ++s) a += slab[(size_t)s * rows * width + i];
        a *= scale[1];
    }
    ((typename Elem<DT>::type*)out)[n * out_stride + m] = from_float<DT>(a);
}

}  // namespace q1head
