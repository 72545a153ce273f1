// q1head_calls.hpp - host side of the wide categorical head: which kernels of q1head.hpp run on which tiles, in which workspace.  Included by the translation units of the three element
// types (q1env_head_f32 / _bf16 / _f16.hip), which are compiled side by side, and by q1env_head.hip for the sizes.
#pragma once
#include "q1env_host.hpp"
#include "q1head.hpp"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace q1head {
namespace {

// of the gradient of one piece of the classes, which is 256 classes at least: beyond 305 000 float32 or 917 000 16-bit rows that is more (6.4 GB at 2^22 float32 rows).
// (Half of it: 15 % slower at 50000 x 256 x 4097 and 4096 x 1024 x 32768, 1 % at 8192 x 2048 x 131072.)
constexpr uint64_t PIECE_BYTES = 448ull << 20;
// of the laid-out weights of one piece.  float32 always needs them: a piece of 96 MiB costs 10 to 20 % (1578 x 1344 x 16658: 2115 us against 1726, 64 x 1024 x 50000 forward 238 against 180); 16-bit
// weights only where they are not aligned
constexpr uint64_t laid_bytes(int dt) { return dt == 0 ? 448ull << 20 : 160ull << 20; }
constexpr int64_t MAX_ROWS = 1 << 22, MAX_WIDTH = 1 << 16, MAX_CLASSES = 1 << 22;
constexpr int64_t PIECE_STEP = 256;                // pieces are whole tiles of every configuration
// A launch holds fewer than 2^32 threads.  Tiles whose grid would hold more than half of that are not taken (a quarter for each of the two backward products, which may share a launch), pieces are cut
// so that Large's always fit, and what only streams goes out in several launches.
constexpr int64_t MOST_THREADS = 1ll << 31;

typedef Config<256, 256, 2, 4, 64, 2> Large;           // 128 KB of LDS: one workgroup of eight waves per CU
typedef Config<128, 128, 2, 2, 64, 2> Middle;          // 64 KB: two workgroups of four waves per CU, one computes while the other waits
typedef Config<128, 256, 2, 4, 32, 3, 4> Pair;         // 77 KB: two workgroups of eight waves per CU, one's epilogue beside the other's products; for logits of 16-bit types with a short k
typedef Config<64, 64, 2, 2, 64, 4> Small;         // where Middle's tiles would leave most CUs idle: 64 KB, four steps in flight
typedef Config<128, 64, 4, 1, 64, 3> Few;              // up to 64 rows: 72 KB, two workgroups per CU
typedef Config<128, 32, 4, 1, 64, 4> Fewest;           // up to 32 rows: 80 KB, two workgroups per CU

int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return div_up(a, b) * b; }
uint64_t aligned(uint64_t x) { return (x + 255) & ~255ull; }
size_t elem_size(int dt) { return dt == F32 ? 4 : 2; }
int planes_of(int dt) { return dt == F32 ? 3 : 1; }

// the forward pass's results as the backward pass reads them (q1env_head_state_bytes)
struct State {
    float *top, *rest, *entropy, *each;
    int64_t* target;
    uint8_t* live;
    uint64_t* bits;
    static uint64_t bytes(int64_t n) { return 3 * aligned(4 * n) + aligned(8 * n) + aligned(n) + aligned(8 * div_up(n, 64)) + 256; }
    State(void* p, int64_t n) {
        char* c = (char*)p;
        top = (float*)c; c += aligned(4 * n);
        rest = (float*)c; c += aligned(4 * n);
        entropy = (float*)c; c += aligned(4 * n);
        target = (int64_t*)c; c += aligned(8 * n);
        live = (uint8_t*)c; c += aligned(n);
        bits = (uint64_t*)c; c += aligned(8 * div_up(n, 64));
        each = (float*)c;
    }
};

enum Size { LARGE, MIDDLE, SMALL, PAIR, FEW, FEWEST };
int64_t bm_of(Size s) { return s == LARGE ? 256 : s == SMALL ? 64 : 128; }
int64_t bn_of(Size s) { return s == LARGE || s == PAIR ? 256 : s == MIDDLE ? 128 : s == FEWEST ? 32 : 64; }

// The tile of a product of m x n results with k terms, and into how many parts its sum is split, by what it should take in nanoseconds.  One round of Large workgroups (256,
// one per CU) was measured at 31 ns per term of k (1075 TFLOP/s), one of Middle (512, two per CU) at 18 (930), of Pair (512) at 36; Start is what a round costs besides, prologue and epilogue:
// 50176 x 256 x 4352 (whole tiles), each kernel alone in a loop, takes 164 / 189 / 151 us of statistics and 250 / 294 / 219 of gradients in Large / Middle / Pair, 4096 x 1024 x 32768 282 / 356 / 331 of statistics.  The slabs of a split sum
// are written and read once at 4.5 TB/s.
struct Start { double large, middle, pair; };          // nanoseconds; pair 0: not for this product
constexpr Start STATISTICS{4500.0, 2600.0, 2400.0}, GRADIENT{11500.0, 6800.0, 7600.0}, PRODUCT{4000.0, 3000.0, 0.0};
// `split` false: one part only
struct Shape { Size size; int parts; int64_t len; };
Shape shape_of(int64_t m, int64_t n, int64_t k, int products, bool split, const Start& starts, bool k_major) {
    if (n <= 64 && !k_major) {                        // few rows: 512 workgroups (two per CU), parts of 512 terms at least
        const Size s = n <= 32 ? FEWEST : FEW;
        const int64_t tiles = div_up(m, bm_of(s));
        int64_t parts = split ? std::max<int64_t>(1, std::min(div_up(512, tiles), div_up(k, 512))) : 1;
        const int64_t len = round_up(div_up(k, parts), PART_STEP);
        return Shape{s, (int)div_up(k, len), len};
    }
    Shape best{MIDDLE, 1, round_up(k, PART_STEP)};
    double least = 0.0;
    for (int s = LARGE; s <= PAIR; ++s) {
        if (s == PAIR && (starts.pair == 0.0 || products > 1)) continue;
        const int64_t tiles = div_up(m, bm_of((Size)s)) * div_up(n, bn_of((Size)s)), slots = s == LARGE ? 256 : 512;
        const int64_t threads = s == LARGE || s == PAIR ? 512 : 256, groups_most = (split ? MOST_THREADS / 2 : MOST_THREADS) / threads;
        const double start = s == LARGE ? starts.large : s == MIDDLE ? starts.middle : s == PAIR ? starts.pair : starts.middle / 2;
        const int64_t most = split ? std::min<int64_t>(div_up(k, 256), std::max<int64_t>(1, div_up(4 * slots, tiles))) : 1;
        for (int64_t parts = 1; parts <= most; ++parts) {
            const int64_t len = round_up(div_up(k, parts), PART_STEP), real = div_up(k, len), groups = tiles * real;
            if (groups > groups_most) break;
            // a term of k of one round; of a round that leaves every workgroup a CU to itself
            const double full = s == LARGE ? 31.0 : s == MIDDLE ? 18.0 : s == PAIR ? 36.0 : 9.5, alone = s == LARGE ? 31.0 : s == MIDDLE ? 11.0 : s == PAIR ? 20.0 : 5.0;
            double t = (double)div_up(groups, slots) * ((double)len * products * (groups <= 256 ? alone : full) + start);
            if (real > 1) t += 3000.0 + (double)real * (double)m * (double)n * 8.0 / 4500.0;
            if (least == 0.0 || t < least) { least = t; best = Shape{(Size)s, (int)real, len}; }
        }
    }
    return best;
}

// Both backward products in one launch, dw's workgroups first: the time at which the last of a workgroups of ta and then b of tb ends on `slots` places.
double last_of(int64_t a, double ta, int64_t b, double tb, int64_t slots) {
    const int64_t full = a / slots, late = a % slots;                         // places that are free after `full` rounds, and after one more
    const double t0 = (double)full * ta, t1 = late ? t0 + ta : t0;
    double best = 0.0;
    for (int64_t k = b / slots; b > 0; ++k) {                                 // rounds of b on the early places, or on the late ones: the first that holds all of them
        for (const double t : {t0 + (double)k * tb, t1 + (double)k * tb}) {
            const int64_t on_late = t >= t1 ? (int64_t)((t - t1) / tb + 1e-9) : 0, on_early = (int64_t)((t - t0) / tb + 1e-9);
            if ((slots - late) * on_early + late * on_late >= b && (best == 0.0 || t < best)) best = t;
        }
        if (best > 0.0) break;
    }
    return std::max(t1, best);
}
// Splits both so that the last round comes out even (1003 x 1000 x 50001: 784 workgroups of 16 steps and 16 x 15 of 53 in place of 16 x 16 of 49: the whole call 500 us in place of 516).  Tried around what each would choose alone.
void split_together(Shape& dw, int64_t dw_m, int64_t dw_n, int64_t dw_k, Shape& dh, int64_t dh_m, int64_t dh_n, int64_t dh_k, int products) {
    if (dw.size != dh.size || dw.size > SMALL) return;
    const Size s = dw.size;
    const int64_t slots = s == LARGE ? 256 : 512, ta = div_up(dw_m, bm_of(s)) * div_up(dw_n, bn_of(s)), tb = div_up(dh_m, bm_of(s)) * div_up(dh_n, bn_of(s));
    const double step = (s == LARGE ? 31.0 : s == MIDDLE ? 18.0 : 9.5) * products, start = s == LARGE ? PRODUCT.large : s == MIDDLE ? PRODUCT.middle : PRODUCT.middle / 2;
    auto slabs = [](int64_t parts, int64_t m, int64_t n) { return parts > 1 ? (double)parts * (double)m * (double)n * 8.0 / 4500.0 : 0.0; };
    if ((double)(ta * dw_k + tb * dh_k) * step / (double)slots < 50000.0) return;                       // not worth the search
    double least = 0.0;
    const Shape w0 = dw, h0 = dh;
    for (int64_t p = std::max(1, w0.parts - 3); p <= w0.parts + 3; ++p) {
        const int64_t lw = round_up(div_up(dw_k, p), PART_STEP), rw = div_up(dw_k, lw);
        if (rw != p && p > 1) continue;
        for (int64_t q = std::max(1, h0.parts / 2); q <= 2 * h0.parts + 4; ++q) {
            const int64_t lh = round_up(div_up(dh_k, q), PART_STEP), rh = div_up(dh_k, lh);
            if (rh != q && q > 1) continue;
            const double t = last_of(ta * rw, (double)lw * step + start, tb * rh, (double)lh * step + start, slots) + slabs(rw, dw_m, dw_n) + slabs(rh, dh_m, dh_n);
            if (least == 0.0 || t < least) {
                least = t;
                dw = Shape{s, (int)rw, lw};
                dh = Shape{s, (int)rh, lh};
            }
        }
    }
}

bool in_place(int dt, const void* p, int64_t stride, int64_t width) {       // whether the loads can take an operand as it lies
    return dt != F32 && ((uintptr_t)p & 15) == 0 && stride % 8 == 0 && width % 8 == 0 && stride < (1 << 21);
}

struct Plan {
    int64_t padded;                    // width of laid-out rows
    int64_t piece;                     // classes per piece
    int64_t pieces;
    Size logits, dh, dw;
    int dh_split, dw_split;
    int64_t dh_k, dw_k;                // classes / rows per split
    bool skinny;                       // float32 with at most 32 rows or classes
    bool two;                          // the gradient of 16-bit operands in two pieces
    int64_t tiles;                     // partial statistics per row
    int64_t g_stride, teams;           // skinny: of the gradient's rows; groups of rows
    uint64_t part, own, scale, g, db, dh_slab, dw_slab, h_laid, w_laid;        // byte offsets in the workspace
    uint64_t bytes;
};

// a skinny product's sums: 512 workgroups of four waves, parts of 256 terms at least, 128 parts at most
void skinny_split(int64_t tiles, int64_t k, int& n, int64_t& len) {
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>({div_up(512, tiles), div_up(k, 256), 128}));
    len = round_up(div_up(k, parts), 32);
    n = (int)div_up(k, len);
}

// of the pieces of at most `most` classes that come to `pieces` of them, the size whose 256 x 256 tiles take the fewest rounds over the CUs (4096 x 1024 x 32768 float32: two of 16384 instead of
// 18944 and 13824 take 5200 us instead of 5880; 8192 x 2048 x 131072: four of 28672 and one of 16384 14470, five of 26368 15000)
int64_t even_piece(int64_t most, int64_t pieces, int64_t classes, int64_t rows) {
    if (pieces == 1) return most;
    const int64_t r = div_up(rows, 256), all = div_up(classes, PIECE_STEP), last = most / PIECE_STEP, first = std::min(last, div_up(all, pieces)), step = std::max<int64_t>(1, (last - first) / 64);
    int64_t best = first, least = INT64_MAX;
    for (int64_t c = first; c <= last; c += step) {
        const int64_t whole = all / c, rounds = whole * div_up(c * r, 256) + div_up((all - whole * c) * r, 256);
        if (rounds <= least) { least = rounds; best = c; }                    // (the largest of equals: longer sums in dh)
    }
    return best * PIECE_STEP;
}

// w_in_place / h_in_place: the workspace has to suffice for any address, so its size is asked for with both false
Plan plan_of(int dt, int64_t rows, int64_t width, int64_t classes, bool backward, bool h_in_place, bool w_in_place) {
    Plan p{};
    p.skinny = dt == F32 && width >= 4 && (rows <= 32 || classes <= 32);
    p.two = dt != F32 && rows <= 256;                                         // (gradient_kernel)
    if (p.skinny) h_in_place = w_in_place = true;
    p.padded = round_up(width, 64);
    const int64_t all = round_up(classes, PIECE_STEP);
    int64_t piece = all;
    const int64_t g_pieces = p.two ? 2 : planes_of(dt);                        // of the stored gradient
    const int64_t laid = planes_of(dt) * 2 * p.padded;                        // bytes of a laid-out row
    if (!w_in_place) piece = std::min<int64_t>(piece, std::max<int64_t>(PIECE_STEP, (int64_t)(laid_bytes(dt) / laid) / PIECE_STEP * PIECE_STEP));
    if (backward) piece = std::min<int64_t>(piece, std::max<int64_t>(PIECE_STEP, (int64_t)(PIECE_BYTES / (2 * g_pieces * rows)) / PIECE_STEP * PIECE_STEP));
    piece = std::min<int64_t>(piece, std::max<int64_t>(1, MOST_THREADS / 512 / div_up(rows, 256)) * PIECE_STEP);          // Large: 512 threads to a tile of 256 x 256
    p.pieces = div_up(classes, piece);
    p.piece = piece = even_piece(piece, p.pieces, classes, rows);
    p.pieces = div_up(classes, piece);
    const int products = planes_of(dt) == 3 ? 6 : 1;
    p.logits = shape_of(std::min(piece, classes), rows, width, products, false, backward ? GRADIENT : STATISTICS, false).size;
    if (backward && p.two && (p.logits == LARGE || p.logits == PAIR)) p.logits = MIDDLE;          // (the others' registers do not last for the second piece)
    uint64_t at = 0;
    auto take = [&](uint64_t n) { const uint64_t o = at; at += aligned(n); return o; };
    if (!backward) {
        p.own = take(4 * rows);
        p.tiles = p.skinny ? std::min<int64_t>(div_up(classes, 32), 2048) : div_up(classes, bm_of(p.logits));
        p.part = take(12 * (uint64_t)p.tiles * rows);
    } else if (p.skinny) {
        p.piece = classes;
        p.pieces = 1;
        p.g_stride = round_up(classes, 32);
        p.teams = std::max<int64_t>(1, std::min(div_up(rows, 32), 1024 / std::min<int64_t>(1024, div_up(classes, 32))));
        skinny_split(div_up(width, 128) * div_up(rows, 32), classes, p.dh_split, p.dh_k);
        skinny_split(div_up(width, 128) * div_up(classes, 32), rows, p.dw_split, p.dw_k);
        p.scale = take(256);
        p.g = take(4 * (uint64_t)rows * p.g_stride);
        p.db = take(4 * (uint64_t)p.teams * classes);
        p.dh_slab = take(p.dh_split > 1 ? 4 * (uint64_t)p.dh_split * rows * width : 0);
        p.dw_slab = take(p.dw_split > 1 ? 4 * (uint64_t)p.dw_split * classes * width : 0);
    } else {
        Shape dh = shape_of(width, rows, std::min(piece, classes), products * (p.two ? 2 : 1), true, PRODUCT, false);
        Shape dw = shape_of(width, std::min(piece, classes), rows, products * (p.two ? 2 : 1), true, PRODUCT, true);
        split_together(dw, width, std::min(piece, classes), rows, dh, width, rows, std::min(piece, classes), products * (p.two ? 2 : 1));
        p.dh = dh.size; p.dh_split = dh.parts; p.dh_k = dh.len;
        p.dw = dw.size; p.dw_split = dw.parts; p.dw_k = dw.len;
        p.scale = take(256);
        p.g = take(2 * (uint64_t)g_pieces * rows * piece);
        p.db = take(4 * (uint64_t)div_up(rows, bn_of(p.logits)) * classes);
        p.dh_slab = take(p.dh_split > 1 || p.pieces > 1 ? 4 * (uint64_t)p.dh_split * rows * width : 0);
        p.dw_slab = take(p.dw_split > 1 ? 4 * (uint64_t)p.dw_split * piece * width : 0);
    }
    p.h_laid = take(h_in_place ? 0 : (uint64_t)laid * rows);
    p.w_laid = take(w_in_place ? 0 : (uint64_t)laid * piece);
    p.bytes = at;
    return p;
}

// what a workspace has to hold whatever the operands' addresses and strides are
uint64_t workspace_of(int dt, int64_t rows, int64_t width, int64_t classes, bool backward) {
    uint64_t n = plan_of(dt, rows, width, classes, backward, false, false).bytes;
    if (dt != F32 && width % 8 == 0)                                          // pieces differ: either may need more
        n = std::max(n, plan_of(dt, rows, width, classes, backward, false, true).bytes);
    return n;
}

template <class C, auto KERNEL, typename... A> int go(hipStream_t stream, int device, int64_t workgroups, A... args) {
    if (workgroups <= 0 || workgroups * C::THREADS >= 1ll << 32) return fail(Q1ENV_ERR_INVALID_ARG, "wide categorical head: too many tiles");
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = 1ull << (device & 63);
    if (C::ALL_BYTES > 65536 && (device > 63 || !(done.load(std::memory_order_relaxed) & bit))) {        // more than 64 KB of LDS has to be allowed once per kernel and device
        HIP_TRY(hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, C::ALL_BYTES));
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(KERNEL, dim3((unsigned)workgroups), dim3(C::THREADS), C::ALL_BYTES, stream, args...);
    HIP_TRY(hipGetLastError());
    return 0;
}
#define Q1_TRY(expr) do { if (int rc_ = (expr)) return rc_; } while (0)

struct Where { hipStream_t stream; int device; };

template <class C, int DT> int statistics(const Where& at, Head hd, const Target& target, bool entropy, float* part, float* own) {
    hd.tiles_m = (uint32_t)div_up(hd.c1 - hd.c0, C::BM);
    hd.tiles_n = (uint32_t)div_up(hd.rows, C::BN);
    const int64_t workgroups = (int64_t)hd.tiles_m * hd.tiles_n;
    return entropy ? go<C, statistics_kernel<C, DT, true>>(at.stream, at.device, workgroups, hd, target, hd.c0 / C::BM, part, own)
                   : go<C, statistics_kernel<C, DT, false>>(at.stream, at.device, workgroups, hd, target, hd.c0 / C::BM, part, own);
}
template <class C, int DT, int GP> int gradient(const Where& at, Head hd, const Upstream& up, int64_t piece, const State& st, uint16_t* g, float* db) {
    hd.tiles_m = (uint32_t)div_up(hd.c1 - hd.c0, C::BM);
    hd.tiles_n = (uint32_t)div_up(hd.rows, C::BN);
    const int64_t workgroups = (int64_t)hd.tiles_m * hd.tiles_n, plane = hd.rows * piece;
    const float *top = st.top, *rest = st.rest, *entropy = st.entropy;
    return up.dentropy ? go<C, gradient_kernel<C, DT, GP, true>>(at.stream, at.device, workgroups, hd, up, piece, plane, top, rest, entropy, g, db)
                       : go<C, gradient_kernel<C, DT, GP, false>>(at.stream, at.device, workgroups, hd, up, piece, plane, top, rest, entropy, g, db);
}
// workgroups of a product in C's tiles
template <class C> int64_t tiles_of(Product& pr, int splits) {
    pr.tiles_m = (uint32_t)div_up(pr.width, C::BM);
    pr.tiles_n = (uint32_t)div_up(pr.rows, C::BN);
    return (int64_t)pr.tiles_m * pr.tiles_n * splits;
}
// dw and dh may each be absent (null out)
template <class C, int DT, int GP> int products(const Where& at, Product dw, int dw_split, Product dh, int dh_split, const Upstream& up) {
    const int64_t a = dw.out ? tiles_of<C>(dw, dw_split) : 0, b = dh.out ? tiles_of<C>(dh, dh_split) : 0, padded = b > 0 ? round_up(a, 8) : a;
    return a + b == 0 ? 0 : go<C, products_kernel<C, DT, GP>>(at.stream, at.device, padded + b, dw, dh, up, (uint32_t)a, (uint32_t)padded);
}
template <class C, int DT, int GP> int rows_product(const Where& at, Product dh, int dh_split, const Upstream& up) {
    const int64_t groups = tiles_of<C>(dh, dh_split);
    return go<C, rows_product_kernel<C, DT, GP>>(at.stream, at.device, groups, dh, up);
}

// lays out what has rows, in one launch
template <int DT> int lay_out(const Where& at, Lay a, Lay b, int64_t width, int64_t padded) {
    const int64_t ga = div_up(a.rows * padded, 2048), gb = div_up(b.rows * padded, 2048);
    a.groups = ga;
    for (int64_t from = 0; from < ga + gb; from += MOST_THREADS / 256) {
        hipLaunchKernelGGL((lay_out_kernel<DT>), dim3((unsigned)std::min(ga + gb - from, MOST_THREADS / 256)), dim3(256), 0, at.stream, a, b, width, padded, from);
        HIP_TRY(hipGetLastError());
    }
    return 0;
}
// adds the parts of the sums up
template <int DT> int add_parts(const Where& at, const Finish& fw, const Finish& fh, const FinishBias& fb, const Upstream& up) {
    const int64_t groups = (int64_t)fw.groups + fh.groups + fb.groups;
    for (int64_t from = 0; from < groups; from += MOST_THREADS / 256) {
        hipLaunchKernelGGL((finish_kernel<DT>), dim3((unsigned)std::min(groups - from, MOST_THREADS / 256)), dim3(256), 0, at.stream, fw, fh, fb, up, (uint32_t)from);
        HIP_TRY(hipGetLastError());
    }
    return 0;
}

// an operand of `rows` rows, as it lies or laid out at `laid` (then the rows have been laid out already)
Op rows_op(int dt, bool as_it_lies, const void* p, int64_t stride, int64_t rows, int64_t width, int64_t padded, const void* laid) {
    if (as_it_lies) return Op{(const char*)p, 2 * stride, 0, rows, width, nullptr};
    return Op{(const char*)laid, 2 * padded, 2 * rows * padded, rows, padded, nullptr};
}
// the same memory with the rows as the k of a product
Op turned(const Op& o, const uint64_t* live) { return Op{o.p, o.stride, o.plane, o.k_extent, o.x_extent, live}; }

Skinny skinny_of(const q1env_head& q) {
    return Skinny{(const float*)q.weight_dev, (const float*)q.hidden_dev, (const float*)q.bias_dev, q.weight_stride, q.hidden_stride, q.rows, q.width, q.classes};
}
int skinny_statistics(const Where& at, const Skinny& q, const Target& target, bool entropy, int64_t tiles, float* part, float* own) {
    const dim3 groups((unsigned)(tiles * div_up(q.rows, 32)));
    if (entropy) hipLaunchKernelGGL((skinny_statistics_kernel<true>), groups, dim3(256), 0, at.stream, q, target, (uint32_t)tiles, part, own);
    else hipLaunchKernelGGL((skinny_statistics_kernel<false>), groups, dim3(256), 0, at.stream, q, target, (uint32_t)tiles, part, own);
    HIP_TRY(hipGetLastError());
    return 0;
}
int skinny_gradient(const Where& at, const Skinny& q, const Upstream& up, const State& st, uint32_t teams, float* g, int64_t stride, float* db) {
    const uint32_t groups = (uint32_t)div_up(q.classes, 32);
    const dim3 grid(groups * teams);
    const int64_t* t = st.target;
    const float *top = st.top, *rest = st.rest, *entropy = st.entropy;
    if (up.dentropy) hipLaunchKernelGGL((skinny_gradient_kernel<true>), grid, dim3(256), 0, at.stream, q, up, t, groups, teams, top, rest, entropy, g, stride, db);
    else hipLaunchKernelGGL((skinny_gradient_kernel<false>), grid, dim3(256), 0, at.stream, q, up, t, groups, teams, top, rest, entropy, g, stride, db);
    HIP_TRY(hipGetLastError());
    return 0;
}
int skinny_product(const Where& at, SkinnyProduct q, bool b_k_major, const Upstream& up) {
    q.tiles_m = (uint32_t)div_up(q.m, 128);
    q.tiles_n = (uint32_t)div_up(q.n, 32);
    const bool shared = q.part >= 128;                                        // long sums: four waves to a unit
    const int64_t units = (int64_t)q.tiles_m * q.tiles_n * q.splits, groups = shared ? units : div_up(units, 4);
    if (groups * 256 >= 1ll << 32) return fail(Q1ENV_ERR_INVALID_ARG, "wide categorical head: too many tiles");
    const dim3 g((unsigned)groups), b(256);
    if (b_k_major) {
        if (shared) hipLaunchKernelGGL((skinny_product_kernel<true, true>), g, b, 0, at.stream, q, up);
        else hipLaunchKernelGGL((skinny_product_kernel<true, false>), g, b, 0, at.stream, q, up);
    } else {
        if (shared) hipLaunchKernelGGL((skinny_product_kernel<false, true>), g, b, 0, at.stream, q, up);
        else hipLaunchKernelGGL((skinny_product_kernel<false, false>), g, b, 0, at.stream, q, up);
    }
    HIP_TRY(hipGetLastError());
    return 0;
}

template <int DT>
int forward(const Where& at, const q1env_head& q, int reduction, float* logp, float* entropy, float* loss) {
    const int64_t n = q.rows;
    const int mean = reduction == Q1ENV_REDUCE_MEAN ? 1 : 0;
    State st(q.state_dev, n);
    if (n > 0) {
        const bool hp = in_place(DT, q.hidden_dev, q.hidden_stride, q.width), wp = in_place(DT, q.weight_dev, q.weight_stride, q.width);
        const Plan p = plan_of(DT, n, q.width, q.classes, false, hp, wp);
        char* ws = (char*)q.ws_dev;
        const Target target{q.target_dev, q.target_bits == 64 ? 1 : 0, q.ignore_index, q.classes};
        const Op h = rows_op(DT, hp, q.hidden_dev, q.hidden_stride, n, q.width, p.padded, ws + p.h_laid);
        float *part = (float*)(ws + p.part), *own = (float*)(ws + p.own);
        if constexpr (DT == F32)
            if (p.skinny) {
                const Skinny sk = skinny_of(q);
                Q1_TRY(skinny_statistics(at, sk, target, entropy != nullptr, p.tiles, part, own));
            }
        for (int64_t c0 = 0; c0 < q.classes && !p.skinny; c0 += p.piece) {
            const int64_t c1 = std::min(c0 + p.piece, q.classes);
            const char* w0 = (const char*)q.weight_dev + elem_size(DT) * c0 * q.weight_stride;
            Q1_TRY(lay_out<DT>(at, Lay{q.hidden_dev, q.hidden_stride, hp || c0 > 0 ? 0 : n, nullptr, (uint16_t*)(ws + p.h_laid), 0},
                               Lay{w0, q.weight_stride, wp ? 0 : c1 - c0, nullptr, (uint16_t*)(ws + p.w_laid), 0}, q.width, p.padded));
            const Head hd{rows_op(DT, wp, w0, q.weight_stride, c1 - c0, q.width, p.padded, ws + p.w_laid), h, q.bias_dev, nullptr, n, q.width, q.classes, 0, 0, c0, c1};
            const bool e = entropy != nullptr;
            if (p.logits == LARGE) Q1_TRY((statistics<Large, DT>(at, hd, target, e, part, own)));
            else if (p.logits == MIDDLE) Q1_TRY((statistics<Middle, DT>(at, hd, target, e, part, own)));
            else if (p.logits == PAIR) Q1_TRY((statistics<std::conditional_t<DT == F32, Middle, Pair>, DT>(at, hd, target, e, part, own)));          // (never float32)
            else if (p.logits == SMALL) Q1_TRY((statistics<Small, DT>(at, hd, target, e, part, own)));
            else if (p.logits == FEW) Q1_TRY((statistics<Few, DT>(at, hd, target, e, part, own)));
            else Q1_TRY((statistics<Fewest, DT>(at, hd, target, e, part, own)));
        }
        const bool tall = p.tiles > 64 && n <= 4096;                          // many tiles of few rows
        float* here = n <= (tall ? 16 : 64) ? loss : nullptr;                 // one workgroup joins all the rows: it has the loss too
        if (tall)
            hipLaunchKernelGGL((join_kernel<16>), dim3((unsigned)div_up(n, 16)), dim3(1024), 0, at.stream, part, own, target, n, (int)p.tiles, entropy ? 1 : 0, logp, entropy, st.entropy,
                               st.top, st.rest, st.target, st.live, st.bits, mean, here, st.each);
        else
            hipLaunchKernelGGL((join_kernel<64>), dim3((unsigned)div_up(n, 64)), dim3(1024), 0, at.stream, part, own, target, n, (int)p.tiles, entropy ? 1 : 0, logp, entropy, st.entropy,
                               st.top, st.rest, st.target, st.live, st.bits, mean, here, st.each);
        HIP_TRY(hipGetLastError());
        if (here) return Q1ENV_OK;
    }
    if (loss) {
        hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(1024), 0, at.stream, logp, st.live, n, mean, loss, st.each);
        HIP_TRY(hipGetLastError());
    }
    return Q1ENV_OK;
}

template <int DT, int GP>
int backward(const Where& at, const q1env_head& q, const Plan& p, bool hp, bool wp, Upstream up, void* dh, int64_t dh_stride, void* dw, int64_t dw_stride, void* db) {
    const int64_t n = q.rows, v = q.classes, d = q.width;
    State st(q.state_dev, n);
    char* ws = (char*)q.ws_dev;
    float* db_part = db ? (float*)(ws + p.db) : nullptr;
    up.each = up.dloss ? st.each : nullptr;
    up.f16 = DT == F16;
    if (DT == F16 && !up.dloss) {
        hipLaunchKernelGGL(scale_kernel, dim3(1), dim3(1024), 0, at.stream, up, st.live, n, (float*)(ws + p.scale));
        HIP_TRY(hipGetLastError());
        up.table = (const float*)(ws + p.scale);
    }
    auto four = [&](const void* out, int64_t stride) { return d % 4 == 0 && stride % 4 == 0 && (uintptr_t)out % (4 * elem_size(DT)) == 0; };
    if constexpr (DT == F32)
        if (p.skinny) {
            float *g = (float*)(ws + p.g), *hs = p.dh_split > 1 ? (float*)(ws + p.dh_slab) : nullptr, *ss = p.dw_split > 1 ? (float*)(ws + p.dw_slab) : nullptr;
            const Skinny sk = skinny_of(q);
            const uint32_t teams = (uint32_t)p.teams;
            Q1_TRY(skinny_gradient(at, sk, up, st, teams, g, p.g_stride, db_part));
            if (dw)
                Q1_TRY(skinny_product(at, SkinnyProduct{sk.h, g, sk.h_stride, p.g_stride, st.live, d, v, n, p.dw_k, 0, 0, (uint32_t)p.dw_split, ss ? ss : (float*)dw, dw_stride, ss != nullptr,
                                                        nullptr}, true, up));
            if (dh)
                Q1_TRY(skinny_product(at, SkinnyProduct{sk.w, g, sk.w_stride, p.g_stride, nullptr, d, n, v, p.dh_k, 0, 0, (uint32_t)p.dh_split, hs ? hs : (float*)dh, dh_stride, hs != nullptr,
                                                        st.live}, false, up));
            Finish fw{ss, p.dw_split, v, d, nullptr, dw, dw_stride, four(dw, dw_stride) ? 1 : 0, dw && ss ? (uint32_t)div_up(v * d, 1024) : 0};
            Finish fh{hs, p.dh_split, n, d, st.live, dh, dh_stride, four(dh, dh_stride) ? 1 : 0, dh && hs ? (uint32_t)div_up(n * d, 1024) : 0};
            FinishBias fb{db_part, v, (int)p.teams, db, db ? (uint32_t)div_up(v, 64) : 0};
            return add_parts<DT>(at, fw, fh, fb, up);
        }
    const Op h = rows_op(DT, hp, q.hidden_dev, q.hidden_stride, n, d, p.padded, ws + p.h_laid);
    uint16_t* g = (uint16_t*)(ws + p.g);
    float *dh_slab = p.dh_split > 1 || p.pieces > 1 ? (float*)(ws + p.dh_slab) : nullptr, *dw_slab = p.dw_split > 1 ? (float*)(ws + p.dw_slab) : nullptr;
    const int64_t es = (int64_t)elem_size(DT);
    // 16-byte stores of a result: address, stride, and for 16-bit types whole chunks of 8 columns; four values at a time from a slab
    auto wide = [&](const void* out, int64_t stride, const float* slab) { return slab ? d % 4 == 0 : ((uintptr_t)out & 15) == 0 && stride * es % 16 == 0 && (es == 4 || d % 8 == 0); };
    for (int64_t c0 = 0; c0 < v; c0 += p.piece) {
        const int64_t c1 = std::min(c0 + p.piece, v), len = c1 - c0;
        const bool last = c1 == v;
        const char* w0 = (const char*)q.weight_dev + es * c0 * q.weight_stride;
        Q1_TRY(lay_out<DT>(at, Lay{q.hidden_dev, q.hidden_stride, hp || c0 > 0 ? 0 : n, st.live, (uint16_t*)(ws + p.h_laid), 0},
                           Lay{w0, q.weight_stride, wp ? 0 : len, nullptr, (uint16_t*)(ws + p.w_laid), 0}, d, p.padded));
        const Op w = rows_op(DT, wp, w0, q.weight_stride, len, d, p.padded, ws + p.w_laid);
        const Head hd{w, h, q.bias_dev, st.target, n, d, v, 0, 0, c0, c1};
        if (p.logits == LARGE) Q1_TRY((gradient<std::conditional_t<GP == 2, Middle, Large>, DT, GP>(at, hd, up, p.piece, st, g, db_part)));          // (two pieces: never LARGE)
        else if (p.logits == MIDDLE) Q1_TRY((gradient<Middle, DT, GP>(at, hd, up, p.piece, st, g, db_part)));
        else if (p.logits == PAIR) Q1_TRY((gradient<std::conditional_t<GP == 1, Pair, Middle>, DT, GP>(at, hd, up, p.piece, st, g, db_part)));          // (one piece: never float32)
        else if (p.logits == SMALL) Q1_TRY((gradient<Small, DT, GP>(at, hd, up, p.piece, st, g, db_part)));
        else if (p.logits == FEW) Q1_TRY((gradient<Few, DT, GP>(at, hd, up, p.piece, st, g, db_part)));
        else Q1_TRY((gradient<Fewest, DT, GP>(at, hd, up, p.piece, st, g, db_part)));
        const Op gr{(const char*)g, 2 * p.piece, 2 * n * p.piece, n, round_up(len, PART_STEP), nullptr};         // [row][class of the piece]
        Op gt = turned(gr, nullptr);
        gt.x_extent = round_up(len, 8);
        Product pw{turned(h, hp ? st.bits : nullptr), gt, n, p.dw_k, len, d, 0, 0, dw ? (char*)dw + es * c0 * dw_stride : nullptr, dw_stride, 0, dw_slab, 0, nullptr};
        Product ph{turned(w, nullptr), gr, len, p.dh_k, n, d, 0, 0, dh, dh_stride, 0, dh_slab, c0 > 0 ? 1 : 0, st.live};
        pw.vec = wide(pw.out, dw_stride, dw_slab);
        ph.vec = wide(dh, dh_stride, dh_slab);
        const Product none{};
        const bool together = p.dw == p.dh && dw && dh;
        if (dw) {
            const Product& with = together ? ph : none;
            if (p.dw == LARGE) Q1_TRY((products<Large, DT, GP>(at, pw, p.dw_split, with, p.dh_split, up)));
            else if (p.dw == MIDDLE) Q1_TRY((products<Middle, DT, GP>(at, pw, p.dw_split, with, p.dh_split, up)));
            else Q1_TRY((products<Small, DT, GP>(at, pw, p.dw_split, with, p.dh_split, up)));
        }
        if (dh && !together) {
            if (p.dh == LARGE) Q1_TRY((products<Large, DT, GP>(at, none, 0, ph, p.dh_split, up)));
            else if (p.dh == MIDDLE) Q1_TRY((products<Middle, DT, GP>(at, none, 0, ph, p.dh_split, up)));
            else if (p.dh == SMALL) Q1_TRY((products<Small, DT, GP>(at, none, 0, ph, p.dh_split, up)));
            else if (p.dh == FEW) Q1_TRY((rows_product<Few, DT, GP>(at, ph, p.dh_split, up)));
            else Q1_TRY((rows_product<Fewest, DT, GP>(at, ph, p.dh_split, up)));
        }
        Finish fw{dw_slab, p.dw_split, len, d, nullptr, pw.out, dw_stride, four(pw.out, dw_stride) ? 1 : 0, dw && dw_slab ? (uint32_t)div_up(len * d, 1024) : 0};
        Finish fh{dh_slab, p.dh_split, n, d, st.live, dh, dh_stride, four(dh, dh_stride) ? 1 : 0, dh && dh_slab && last ? (uint32_t)div_up(n * d, 1024) : 0};
        FinishBias fb{db_part, v, (int)div_up(n, bn_of(p.logits)), db, db && last ? (uint32_t)div_up(v, 64) : 0};
        Q1_TRY(add_parts<DT>(at, fw, fh, fb, up));
    }
    return Q1ENV_OK;
}

template <int DT>
int backward_of(const Where& at, const q1env_head& q, const Upstream& up, void* dh, int64_t dh_stride, void* dw, int64_t dw_stride, void* db) {
    const bool hp = in_place(DT, q.hidden_dev, q.hidden_stride, q.width), wp = in_place(DT, q.weight_dev, q.weight_stride, q.width);
    const Plan p = plan_of(DT, q.rows, q.width, q.classes, true, hp, wp);
    if constexpr (DT != F32)
        if (p.two) return backward<DT, 2>(at, q, p, hp, wp, up, dh, dh_stride, dw, dw_stride, db);
    return backward<DT, Elem<DT>::planes>(at, q, p, hp, wp, up, dh, dh_stride, dw, dw_stride, db);
}

}  // namespace
}  // namespace q1head

// one per element type
#define Q1_HEAD_CALLS(name)                                                                                                                                              \
    Q1_HIDDEN int q1_head_forward_##name(int device, hipStream_t stream, const q1env_head& q, int reduction, float* logp, float* entropy, float* loss);                    \
    Q1_HIDDEN int q1_head_backward_##name(int device, hipStream_t stream, const q1env_head& q, const float* dlogp, const float* dentropy, const float* dloss, void* dh,    \
                                          int64_t dh_stride, void* dw, int64_t dw_stride, void* db);
Q1_HEAD_CALLS(f32)
Q1_HEAD_CALLS(bf16)
Q1_HEAD_CALLS(f16)
#undef Q1_HEAD_CALLS
#define Q1_HEAD_DEFINE(name, DT)                                                                                                                                         \
    int q1_head_forward_##name(int device, hipStream_t stream, const q1env_head& q, int reduction, float* logp, float* entropy, float* loss) {                             \
        return q1head::forward<DT>(q1head::Where{stream, device}, q, reduction, logp, entropy, loss);                                                                     \
    }                                                                                                                                                                     \
    int q1_head_backward_##name(int device, hipStream_t stream, const q1env_head& q, const float* dlogp, const float* dentropy, const float* dloss, void* dh,              \
                                int64_t dh_stride, void* dw, int64_t dw_stride, void* db) {                                                                                \
        return q1head::backward_of<DT>(q1head::Where{stream, device}, q, q1head::Upstream{dlogp, dentropy, dloss, nullptr, nullptr, 0}, dh, dh_stride, dw, dw_stride, db);  \
    }
