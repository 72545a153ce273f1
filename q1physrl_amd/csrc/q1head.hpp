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
// a3 b1, a2 b2; what is dropped is 2^-27 of |a b| typically and 2^-23 at most, under the rounding of the float32 accumulator the products go to.  (The
// float32 matrix instruction runs at 1/16 of the bfloat16 one; six products run at 1/6.)
#pragma once
#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>
#include <type_traits>

namespace q1head {
namespace {                                // every translation unit carries the kernels it launches

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

// a float32 as three bfloat16 pieces, each the nearest to what the ones before leave (a value that would round to infinity keeps the largest finite first piece)
__device__ __forceinline__ uint16_t bf16_bits(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ float bf16_value(uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }
__device__ __forceinline__ uint16_t f16_bits(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
__device__ __forceinline__ float f16_value(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }

__device__ __forceinline__ void three_pieces(float a, uint16_t& p1, uint16_t& p2, uint16_t& p3) {
    p1 = bf16_bits(a);
    if ((p1 & 0x7fff) == 0x7f80 && fabsf(a) < INFINITY) p1 -= 1;
    const float r1 = a - bf16_value(p1);
    p2 = bf16_bits(r1);
    p3 = bf16_bits(r1 - bf16_value(p2));
}

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

// ------------------------------------------------------------------------------------------------------------------------------
// C[m][n] = sum_k A(m, k) B(n, k) on 16-bit operands, a BM x BN tile per workgroup.
//
// An operand lies in memory with k contiguous (KM = false: element (x, k) at p[x stride + k]) or with x contiguous (KM = true: p[k stride + x]).  Both
// kinds travel from memory to LDS without passing through registers (buffer loads with an LDS destination, 16 bytes per lane, 1 KB per
// wave instruction; what lies outside the operand reads as zero by the buffer's bounds check), BK values of k at a time, STAGES tiles in flight:
// the loads of a tile are issued one (two, three) whole steps before its barrier.  The LDS image is linear in the order of the loading lanes, so bank conflicts are
// avoided by permuting which 16-byte chunk a lane asks memory for:
//   KM = false: rows of 2 BK bytes; chunk c of row x sits at c ^ ((x >> 1) & 7) (BK = 64) or c ^ ((x >> 2) & 3) (BK = 32): any 16 lanes of a fragment read (16 rows, one
//               chunk) cover all 64 banks;
//   KM = true:  rows of 2 BM bytes; the 32-byte unit u of row k sits at u ^ (2 (k & 3)) (u ^ (k & 2) in rows of 128 bytes): the transposing read (ds_read_b64_tr_b16: 4 values
//               of k x 16 of x per 16 lanes) touches four rows at four different bank groups.
// Bound (256 x 256 tile, 8 waves of 128 x 64): per step a wave issues 32 matrix instructions of 32 cycles and reads 24 KB of LDS, 75 % of what the LDS delivers in
// that time; a 64 x 64 wave tile would need all of it.
struct Op {
    const char* p;
    int64_t stride;             // bytes from row to row
    int64_t plane;              // bytes from piece to piece (float32 as three bfloat16 pieces)
    int64_t x_extent;           // valid x (KM: a multiple of 8)
    int64_t k_extent;           // valid k (not KM: a multiple of 8)
    const uint64_t* live;       // KM: where set, bit k of the words says whether row k counts (rows that do not are zero whatever memory holds)
};

template <int BM_, int BN_, int WM_, int WN_, int BK_, int STAGES_, int PER_SIMD_ = 1> struct Config {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, BK = BK_, STAGES = STAGES_;
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, PER_SIMD = PER_SIMD_;          // PER_SIMD: waves the registers have to suffice for
    static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;             // 32 x 32 tiles per wave
    static constexpr int LA = BM * BK / 512 / WAVES, LB = BN * BK / 512 / WAVES;         // load instructions per wave and stage
    static constexpr int A_BYTES = BM * BK * 2, STAGE_BYTES = (BM + BN) * BK * 2, LDS_BYTES = STAGES * STAGE_BYTES;
    // what the epilogue over logits wants of every row, behind the stages; not where two workgroups fill the CU's LDS already (they hide each other's loads)
    static constexpr bool KEEPS_ROWS = 2 * LDS_BYTES != 163840;
    static constexpr int ALL_BYTES = LDS_BYTES + (KEEPS_ROWS ? 20 * BN : 0);
    static_assert(BK == 32 || BK == 64, "the LDS image's permutations");
    static_assert(LA * WAVES * 512 == BM * BK && LB * WAVES * 512 == BN * BK && TM >= 1 && TN >= 1, "whole load instructions per wave");
    static_assert(STAGES >= 2 && (STAGES - 1) * (LA + LB) < 64 && ALL_BYTES <= 163840, "vmcnt; LDS of a CU");
};
constexpr int PART_STEP = 64;               // parts of a split sum are whole steps of every configuration (and whole words of `live`)

typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((address_space(3))) char lds_char;
constexpr uint32_t OUTSIDE = 0x80000000u;                                   // the resource's size: an offset from here on reads zero

// size: the bytes from base on that may be read; an offset from there on reads zero
__device__ __forceinline__ void load_to_lds(const char* base, uint32_t size, uint32_t offset, uint32_t lds) {
    const uint64_t a = (uint64_t)base;
    auto uniform = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };      // (all of it is; the resource has to sit in scalar registers)
    const u32x4 rsrc = {uniform((uint32_t)a), uniform((uint32_t)(a >> 32) & 0xffffu), uniform(size), 0x00020000u};
    // (no result registers: what the instruction writes is LDS, waited for with vmcnt before the barrier in front of its use)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(uniform(lds)), "v"(offset), "s"(rsrc) : "memory", "m0");
}
template <int N> __device__ __forceinline__ void wait_loads() {             // all but the N youngest loads have landed, and this wave's LDS reads are done
    static_assert(N < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int XT> __device__ __forceinline__ int unit_flip(int k) { return XT >= 128 ? 2 * (k & 3) : k & 2; }

// The loading side of one operand: XT values of x per tile, COUNT load instructions per wave, each of ROWS rows of the tile.  What a step costs besides the loads is scalar and little
// (130 scalar instructions a step took a fifth of the whole product's time): a lane's offsets stay, the step's address moves; rows past the end of k, and steps past it, lie outside
// the resource and read zero.
template <int XT, int BK, int COUNT, bool KM, bool LIVE> struct Feed {
    static constexpr int ROWS = KM ? 512 / XT : 512 / BK;
    uint32_t off[COUNT];        // byte offset of this lane's chunk in the tile, OUTSIDE if its x is
    int q8[2];                  // not KM: the chunk's k within the step, of even and odd loads
    const char* at;             // the tile at the next step
    int left;                   // of k from the next step on
    uint32_t stride;
    __device__ __forceinline__ void init(const Op& o, int64_t x0, int64_t k0, int wave, int lane) {
        constexpr int PER = KM ? XT / 8 : BK / 8;                            // 16-byte chunks of a row
        const int r = lane / PER, c = lane % PER;
        stride = (uint32_t)o.stride;
#pragma unroll
        for (int j = 0; j < COUNT; ++j) {
            const int row = ROWS * (wave * COUNT + j) + r;
            if constexpr (!KM) {
                const int q = c ^ (BK == 64 ? (row >> 1) & 7 : (row >> 2) & 3);
                off[j] = x0 + row < o.x_extent ? (uint32_t)row * stride + 16 * q : OUTSIDE;
                if (j < 2) q8[j] = 8 * q;
            } else {
                const int x = 8 * (2 * ((c >> 1) ^ unit_flip<XT>(row)) + (c & 1));
                off[j] = x0 + x < o.x_extent ? (uint32_t)row * stride + 2 * x : OUTSIDE;
            }
        }
        if constexpr (COUNT == 1) q8[1] = q8[0];
        at = o.p + (KM ? 2 * x0 + k0 * o.stride : x0 * o.stride + 2 * k0);
        left = (int)(o.k_extent - k0);
    }
    // issues the loads of the next step (its piece `plane`) into the LDS bytes from `lds` on; k0: its first k
    __device__ __forceinline__ void issue(const Op& o, int plane, int64_t k0, uint32_t lds, int wave, int lane) const {
        const char* b = at + plane * o.plane;
        const uint32_t size = KM ? (left >= BK ? OUTSIDE : left > 0 ? (uint32_t)left * stride : 0u) : (left > 0 ? OUTSIDE : 0u);
        uint64_t live = ~0ull;
        if constexpr (LIVE)
            if (o.live && left > 0) live = o.live[k0 / 64] >> (k0 % 64);
        lds += 1024u * (uint32_t)(wave * COUNT);
        if (!KM && left < BK) {                                              // the step that k ends in
#pragma unroll
            for (int j = 0; j < COUNT; ++j) load_to_lds(b, size, q8[j & 1] < left ? off[j] : OUTSIDE, lds + 1024u * j);
        } else {
#pragma unroll
            for (int j = 0; j < COUNT; ++j) {
                uint32_t f = off[j];
                if constexpr (LIVE) f = (live >> (ROWS * (wave * COUNT + j) + lane / (XT / 8))) & 1 ? f : OUTSIDE;
                load_to_lds(b, size, f, lds + 1024u * j);
            }
        }
    }
    __device__ __forceinline__ void advance() {
        at += KM ? (uint64_t)stride * BK : 2 * BK;
        left -= BK;
    }
};

template <class C> struct Acc { f32x16 t[C::TM][C::TN]; };        // lane l: column n = l % 32, register r: row m = 8 (r / 4) + 4 (l / 32) + r % 4

template <class C> __device__ __forceinline__ void clear(Acc<C>& acc) {
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc.t[i][j][r] = 0.0f;
}

// acc += the product of operands in AP and BP pieces.  The products of the pieces (six for float32; two where only the gradient has a second piece) follow each other within every step
// of k, so that a piece's tile is still near when it is asked for again.
// A step's fragments are read one quarter ahead of their use, the last quarter's and the next step's first on either side of the one barrier: the matrix
// instructions behind it have their operands already.  A slot is free at that barrier (its last fragments are in registers), so STAGES steps are in flight.
// `meanwhile` runs when the first steps' loads are under way: it gives acc its first values, and what it loads arrives with them.
template <class C, int DT, int AP, int BP, bool AK, bool BKM, typename F>
__device__ __forceinline__ void gemm_tile(const Op& a, const Op& b, int64_t m0, int64_t n0, int64_t k_begin, int64_t k_end, Acc<C>& acc, char* lds_generic, F&& meanwhile) {
    static_assert((AP == 1 && (BP == 1 || BP == 2)) || (AP == 3 && BP == 3), "pieces of the operands");
    constexpr int SEGS = AP == 3 ? 6 : BP;
    lds_char* lds = (lds_char*)lds_generic;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = (wave % C::WM) * (C::TM * 32), wn = (wave / C::WM) * (C::TN * 32);
    constexpr int BK = C::BK, QUARTERS = BK / 16;                            // of a step: 16 values of k each, one matrix instruction deep
    Feed<C::BM, BK, C::LA, AK, AK && BKM && AP == 1> fa;                        // (hidden rows as k: rows that do not count)
    Feed<C::BN, BK, C::LB, BKM, false> fb;
    fa.init(a, m0, k_begin, wave, lane);
    fb.init(b, n0, k_begin, wave, lane);
    const int steps = k_end > k_begin ? (int)((k_end - k_begin + BK - 1) / BK) * SEGS : 0;
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds;

    int64_t issue_k = k_begin;                                               // of the next step to be issued
    int issue_seg = 0;
    auto issue = [&](int slot) {
        int pa = 0, pb = 0;
        if constexpr (AP == 3) {                                             // (1,1) (0,2) (2,0) (0,1) (1,0) (0,0)
            pa = (0x010201 >> (4 * issue_seg)) & 15;
            pb = (0x001021 >> (4 * issue_seg)) & 15;
        } else if constexpr (BP == 2)
            pb = 1 - issue_seg;
        fa.issue(a, pa, issue_k, lds0 + (uint32_t)slot * C::STAGE_BYTES, wave, lane);
        fb.issue(b, pb, issue_k, lds0 + (uint32_t)slot * C::STAGE_BYTES + C::A_BYTES, wave, lane);
        if (SEGS == 1 || ++issue_seg == SEGS) {
            issue_seg = 0;
            issue_k += BK;
            fa.advance();
            fb.advance();
        }
    };

    // fragment addresses.  not KM: row x, chunk 2 kt + (lane >> 5) of the step; KM: rows 16 kt + 8 (lane >> 5) + 4 h + (s >> 2), unit of x
    uint32_t ra[AK ? C::TM : QUARTERS], rb[BKM ? C::TN : QUARTERS];
    const int s = lane & 15, row = lane & 31, permuted = BK == 64 ? row >> 1 & 7 : row >> 2 & 3;
    if constexpr (!AK) {
#pragma unroll
        for (int kt = 0; kt < QUARTERS; ++kt) ra[kt] = (wm + row) * (2 * BK) + ((2 * kt + (lane >> 5)) ^ permuted) * 16;
    } else {
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
            ra[i] = (8 * (lane >> 5) + (s >> 2)) * (2 * C::BM) + (((wm + 32 * i) / 16 + ((lane >> 4) & 1)) ^ unit_flip<C::BM>(s >> 2)) * 32 + (s & 3) * 8;
    }
    if constexpr (!BKM) {
#pragma unroll
        for (int kt = 0; kt < QUARTERS; ++kt) rb[kt] = C::A_BYTES + (wn + row) * (2 * BK) + ((2 * kt + (lane >> 5)) ^ permuted) * 16;
    } else {
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
            rb[j] = C::A_BYTES + (8 * (lane >> 5) + (s >> 2)) * (2 * C::BN) + (((wn + 32 * j) / 16 + ((lane >> 4) & 1)) ^ unit_flip<C::BN>(s >> 2)) * 32 + (s & 3) * 8;
    }
    auto transposed = [&](uint32_t at, int row_bytes) {
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + at));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + at + 4 * row_bytes));
        const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
        return u32x4{l2[0], l2[1], h2[0], h2[1]};
    };
    u32x4 x[2][C::TM], y[2][C::TN];                                          // fragments: [quarter & 1]
    auto fetch = [&](uint32_t at, int kt) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
            if constexpr (!AK) x[kt & 1][i] = *(__attribute__((address_space(3))) u32x4*)(lds + at + ra[kt] + 64 * BK * i);
            else x[kt & 1][i] = transposed(at + ra[i] + kt * 16 * 2 * C::BM, 2 * C::BM);
        }
#pragma unroll
        for (int j = 0; j < C::TN; ++j) {
            if constexpr (!BKM) y[kt & 1][j] = *(__attribute__((address_space(3))) u32x4*)(lds + at + rb[kt] + 64 * BK * j);
            else y[kt & 1][j] = transposed(at + rb[j] + kt * 16 * 2 * C::BN, 2 * C::BN);
        }
    };
    auto multiply = [&](int kt) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
            for (int j = 0; j < C::TN; ++j) acc.t[i][j] = mfma<DT>(x[kt & 1][i], y[kt & 1][j], acc.t[i][j]);
    };
    // the reads of the next quarter go between the matrix instructions of this one, so that neither waits for the other
    auto interleave = [&]() {
        constexpr int READS = C::TM * (AK ? 2 : 1) + C::TN * (BKM ? 2 : 1), MM = C::TM * C::TN, PER = (READS + MM - 1) / MM;
#pragma unroll
        for (int i = 0; i < MM; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);             // LDS reads
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);               // matrix instructions
        }
    };
#pragma unroll
    for (int g = 0; g < C::STAGES; ++g) issue(g);                            // (steps past the end read zeros: nothing below depends on how many there are)
    meanwhile();
    wait_loads<(C::STAGES - 1) * (C::LA + C::LB)>();
    barrier();
    fetch(0, 0);
    int slot = 0;
    uint32_t at = 0;
#pragma unroll 1
    for (int t = 0; t < steps; ++t) {
#pragma unroll
        for (int kt = 0; kt + 1 < QUARTERS; ++kt) {
            if (kt > 0) __builtin_amdgcn_sched_barrier(0);
            fetch(at, kt + 1);
            multiply(kt);
            interleave();
        }
        wait_loads<(C::STAGES - 2) * (C::LA + C::LB)>();                      // the next step has landed ...
        barrier();                                                           // ... for every wave, and this step's slot has been read
        issue(slot);
        slot = slot == C::STAGES - 1 ? 0 : slot + 1;
        at = (uint32_t)slot * C::STAGE_BYTES;
        fetch(at, 0);
        multiply(QUARTERS - 1);
        interleave();
        __builtin_amdgcn_sched_barrier(0);
    }
    wait_loads<0>();
    barrier();                                                               // the LDS is free again
}

// Workgroup -> tile.  Workgroups are dealt to the eight XCDs in turn, each with an L2 of its own: XCD x takes the x-th eighth of the tiles, and within it tiles go
// in bands of GROUP tiles of n, so that the workgroups that run at one time on one XCD share their operands' tiles on both sides.
__device__ __forceinline__ void tile_of(uint32_t id, uint32_t total, uint32_t tiles_m, uint32_t tiles_n, uint32_t& tm, uint32_t& tn, uint32_t& z) {
    constexpr uint32_t GROUP = 4;
    const uint32_t q = total / 8, r = total % 8, x = id % 8, i = id / 8;
    uint32_t t = x * q + (x < r ? x : r) + i;
    const uint32_t plane = tiles_m * tiles_n;
    z = t / plane;
    t -= z * plane;
    const uint32_t band = t / (GROUP * tiles_m), first = band * GROUP, height = tiles_n - first < GROUP ? tiles_n - first : GROUP;
    t -= band * GROUP * tiles_m;
    tn = first + t % height;
    tm = t / height;
}

// ------------------------------------------------------------------------------------------------------------------------------
// Operands that the loads above cannot take as they lie (float32; a width that is not a multiple of 8, addresses or strides that are not multiples of 16 bytes) are laid out
// first: [piece][row][padded], padded = width rounded up to 64 with zeros; rows that do not count are zero.
// Bound: memory (32768 + 1441 float32 rows of 256: 16 us for 35 MB read and 53 written, 5.4 TB/s).
struct Lay {
    const void* src;
    int64_t stride, rows;             // elements
    const uint8_t* live;
    uint16_t* out;
    int64_t groups;                   // workgroups of 2048 values
};
template <int DT>
__global__ void __launch_bounds__(256) lay_out_kernel(Lay first, Lay second, int64_t width, int64_t padded, int64_t from) {
    const int64_t group = from + blockIdx.x;                                  // (from: of a launch that is not the first)
    const bool one = group < first.groups;
    const Lay& l = one ? first : second;
    const int64_t i = ((one ? group : group - first.groups) * 256 + threadIdx.x) * 8;
    if (i >= l.rows * padded) return;
    const int64_t r = i / padded, k = i - r * padded;
    uint16_t q[Elem<DT>::planes][8];
    const bool on = !l.live || l.live[r];
    const typename Elem<DT>::type* p = (const typename Elem<DT>::type*)l.src + r * l.stride + k;
    typename Elem<DT>::type v[8];
    if (on && k + 8 <= width) __builtin_memcpy(v, p, sizeof v);
    else
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = on && k + j < width ? p[j] : (typename Elem<DT>::type)0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (DT == F32) three_pieces(v[j], q[0][j], q[1][j], q[2][j]);
        else q[0][j] = v[j];
    }
#pragma unroll
    for (int z = 0; z < Elem<DT>::planes; ++z) __builtin_memcpy(l.out + z * l.rows * padded + i, q[z], 16);
}

// the classes as the caller gave them
struct Target {
    const void* p;
    int wide;                        // int64 (else int32)
    int64_t ignore, classes;
    __device__ __forceinline__ int64_t of(int64_t n) const {                // -1: ignored, -2: no such class
        const int64_t t = wide ? ((const int64_t*)p)[n] : (int64_t)((const int32_t*)p)[n];
        return t == ignore ? -1 : (t < 0 || t >= classes ? -2 : t);
    }
};

// what a launch over logit tiles knows of the head
struct Head {
    Op w, h;                         // A: weight (m = class), B: hidden (n = row)
    const void* bias;
    const int64_t* target;           // as join_kernel wrote them (backward)
    int64_t rows, width, classes;
    uint32_t tiles_m, tiles_n;       // of this launch
    int64_t c0, c1;                  // the classes of this launch
};

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// A probability below 2^NOTHING is zero in float32 (the smallest value is 2^-149).  Its logarithm is held to that in the entropy's gradient, where it is multiplied by an upstream value before the
// probability: a class at -inf, or at the type's lowest value, gives 0 x a finite factor.
constexpr float NOTHING = -160.0f;
// Rows whose largest logit lies within this of zero take l log2(e) - m log2(e) as one fma on the rounded m log2(e) (and on the rounded log-sum-exp in the gradient: 2^-17 at most, 5e-6 of a
// probability).  Farther out (masks of the type's lowest value, -1e9, rows that have nothing else) that rounding would be all that is left: there m is subtracted first.
constexpr float NEAR = 128.0f;

// Statistics of a set of classes: the largest logit m, s = sum 2^x and u = sum x 2^x over x = (l - m) log2(e).  One fused multiply-add and one hardware exponential per logit.
struct Stat { float m, s, u; };
__device__ __forceinline__ Stat joined(const Stat& a, const Stat& b) {
    const float m = fmaxf(a.m, b.m);
    // a set of classes at -inf has m = -inf, s = u = 0 and counts nothing; a difference is kept where 0 x (difference x s) is still 0 (masks of the type's lowest value)
    const float da = a.m == -INFINITY ? 0.0f : fmaxf((a.m - m) * LOG2E, -1.0e30f), db = b.m == -INFINITY ? 0.0f : fmaxf((b.m - m) * LOG2E, -1.0e30f);
    const float fa = a.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(da), fb = b.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(db);
    return Stat{m, fa * a.s + fb * b.s, fa * (a.u + da * a.s) + fb * (b.u + db * b.s)};
}

// the sums start from the bias of the classes a lane holds: base + 32 i + 8 r4 + 0 .. 3
template <int DT, class C>
__device__ __forceinline__ void start(Acc<C>& acc, const void* bias, int64_t base, int64_t c1) {
    typedef typename Elem<DT>::type E;
    if (!bias) return clear(acc);
    const E* b = (const E*)bias;
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int64_t m = base + 32 * i + 8 * r4;
            E v[4];
            if (m + 4 <= c1) __builtin_memcpy(v, b + m, sizeof v);
            else
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = m + r < c1 ? b[m + r] : (E)0;
#pragma unroll
            for (int j = 0; j < C::TN; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc.t[i][j][4 * r4 + r] = to_float<DT>(v[r]);
        }
}

// class-tile statistics of each row, and the logit of the row's own class.  The accumulators never leave the registers: one fused multiply-add, one exponential, an addition (and two more
// instructions for the entropy) per logit, then three floats per row and tile.
// Bound: the matrix pipe where k is long (8192 x 2048 x 131072 bfloat16: 3.40 ms, 1290 TFLOP/s, the pipe 67 % busy, no bank conflict; a large library product makes 1225 to 1481); the weights
// where there are few rows (64 x 4096 x 131073: 193 us, 5.6 TB/s); start and epilogue of a tile where k is short (50000 x 256 x 4097: 156 us in a run of passes, 672 TFLOP/s, two workgroups per CU in different
// phases, the pipe 32 % busy; 198 in the first passes of an idle card).
template <class C, int DT, bool ENTROPY>
__global__ void __launch_bounds__(C::THREADS, C::PER_SIMD) statistics_kernel(Head hd, Target target, int64_t tile0, float* __restrict__ part, float* __restrict__ own_logit) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    uint32_t tm, tn, z;
    tile_of(blockIdx.x, gridDim.x, hd.tiles_m, hd.tiles_n, tm, tn, z);
    const int64_t m0 = hd.c0 + (int64_t)tm * C::BM, n0 = (int64_t)tn * C::BN;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave % C::WM) * (C::TM * 32), wn = (wave / C::WM) * (C::TN * 32);
    const int64_t base = m0 + wm + 4 * (lane >> 5);                  // class of the lane's register 0
    Acc<C> acc;
    int* own_of = (int*)(lds + C::LDS_BYTES);                         // the row's own class within the tile, negative: none
    auto own_class = [&](int64_t n) {
        const int64_t t = n < hd.rows ? target.of(n) - m0 : -1;
        return t >= 0 && t < C::BM ? (int)t : -1;
    };
    gemm_tile<C, DT, Elem<DT>::planes, Elem<DT>::planes, false, false>(hd.w, hd.h, m0 - hd.c0, n0, 0, hd.width, acc, lds, [&] {
        start<DT>(acc, hd.bias, base, hd.c1);
        if constexpr (C::KEEPS_ROWS)
            if (threadIdx.x < C::BN) own_of[threadIdx.x] = own_class(n0 + threadIdx.x);
    });
    if (m0 + C::BM > hd.c1) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (base + 32 * i + 8 * (r >> 2) + (r & 3) >= hd.c1)
#pragma unroll
                    for (int j = 0; j < C::TN; ++j) acc.t[i][j][r] = -INFINITY;
    }
    float (*red)[C::BN][3] = (float (*)[C::BN][3])lds;
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
        const int nl = wn + 32 * j + (lane & 31);
        const int rel = (C::KEEPS_ROWS ? own_of[nl] : own_class(n0 + nl)) - wm;
        if (__any(rel >= 0 && rel < C::TM * 32)) {
            const int own = rel >= 4 * (lane >> 5) && rel < C::TM * 32 ? rel - 4 * (lane >> 5) : -1;
            float l = 0.0f;
#pragma unroll
            for (int i = 0; i < C::TM; ++i)
                if (__any(own >= 0 && own >> 5 == i))
#pragma unroll
                    for (int r = 0; r < 16; ++r) l = own == 32 * i + 8 * (r >> 2) + (r & 3) ? acc.t[i][j][r] : l;
            if (own >= 0 && (own & 4) == 0) own_logit[n0 + nl] = l;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, acc.t[i][j][r]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m = mx == -INFINITY ? 0.0f : mx, ref = m * LOG2E;
        float s = 0.0f, u = 0.0f;
        auto add_up = [&](auto near) {
#pragma unroll
            for (int i = 0; i < C::TM; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float d = near ? fmaf(acc.t[i][j][r], LOG2E, -ref) : (acc.t[i][j][r] - m) * LOG2E, e = __builtin_amdgcn_exp2f(d);
                    s += e;
                    if constexpr (ENTROPY) u = fmaf(fmaxf(d, -3.0e38f), e, u);      // a class at -inf adds 0, not 0 x inf
                }
        };
        if (__all(fabsf(m) <= NEAR)) {
            add_up(std::true_type{});
            const float off = fmaf(m, LOG2E, -ref), f = __builtin_amdgcn_exp2f(-off);      // from ref, which was rounded, to m log2(e)
            if constexpr (ENTROPY) u = f * fmaf(-off, s, u);
            s *= f;
        } else
            add_up(std::false_type{});
        s += __shfl_xor(s, 32, 64);
        if constexpr (ENTROPY) u += __shfl_xor(u, 32, 64);
        if (lane < 32) { red[wave % C::WM][nl][0] = mx; red[wave % C::WM][nl][1] = s; red[wave % C::WM][nl][2] = u; }
    }
    __syncthreads();
    for (int nl = threadIdx.x; nl < C::BN; nl += C::THREADS)
        if (n0 + nl < hd.rows) {
            Stat t{red[0][nl][0], red[0][nl][1], red[0][nl][2]};
#pragma unroll
            for (int w = 1; w < C::WM; ++w) t = joined(t, Stat{red[w][nl][0], red[w][nl][1], red[w][nl][2]});
            float* o = part + 3 * (size_t)(tile0 + tm) * hd.rows + n0 + nl;
            o[0] = t.m; o[hd.rows] = t.s; o[2 * hd.rows] = t.u;
        }
}

// Joins the tiles' statistics: R rows per workgroup, 1024 / R lanes take the tiles of a row in turn (four loads of each kind in flight).  The log-sum-exp is kept in its two parts, m and
// log2 s: where m is far from zero their sum would lose the second.  Also leaves what the
// backward pass wants of the classes: -1 / -2 / the class, and the rows that count as bytes and as bits.  R = 64 where there are many rows, 16 where there are many tiles (64 rows
// of 1025 tiles: 21 us with R = 64, 12 with 16).  Bound: latency (8192 rows of 512 tiles: 14 us for 50 MB).
template <int R>
__global__ void __launch_bounds__(1024) join_kernel(const float* __restrict__ part, const float* __restrict__ own_logit, Target target, int64_t rows, int tiles, int with_entropy,
                                                    float* __restrict__ logp, float* __restrict__ entropy, float* __restrict__ entropy_kept, float* __restrict__ top,
                                                    float* __restrict__ rest, int64_t* __restrict__ classes, uint8_t* __restrict__ live, uint64_t* __restrict__ bits, int mean,
                                                    float* __restrict__ loss, float* __restrict__ each) {
    static_assert(R == 64 || R == 16, "the words of bits");
    constexpr int G = 1024 / R;
    __shared__ float red[3][16][R];
    const int r = threadIdx.x % R, g = threadIdx.x / R, wave = threadIdx.x >> 6;
    const int64_t n = (int64_t)blockIdx.x * R + r;
    Stat a{-INFINITY, 0.0f, 0.0f};
    if (n < rows)
        for (int t = g; t < tiles; t += 4 * G) {
            Stat v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float* o = part + 3 * (size_t)(t + G * k) * rows + n;
                v[k] = t + G * k < tiles ? Stat{o[0], o[rows], with_entropy ? o[2 * rows] : 0.0f} : Stat{-INFINITY, 0.0f, 0.0f};
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) a = joined(a, v[k]);
        }
#pragma unroll
    for (int off = R; off < 64; off *= 2) a = joined(a, Stat{__shfl_xor(a.m, off, 64), __shfl_xor(a.s, off, 64), __shfl_xor(a.u, off, 64)});
    if ((threadIdx.x & 63) < R) { red[0][wave][r] = a.m; red[1][wave][r] = a.s; red[2][wave][r] = a.u; }
    __syncthreads();
    if (threadIdx.x >= R) return;
    const int64_t t = n < rows ? target.of(n) : -1;
    const uint64_t word = __ballot(t != -1);
    float lp = 0.0f;
    if (n < rows) {
        for (int k = 1; k < 16; ++k) a = joined(a, Stat{red[0][k][r], red[1][k][r], red[2][k][r]});
        float ls = __log2f(a.s), m = a.m, h = with_entropy ? LN2 * (ls - a.u / a.s) : NAN;
        if (t >= 0) {
            lp = fmaf(-LN2, ls, own_logit[n] - m);
            if (lp == -INFINITY && own_logit[n] != -INFINITY) lp = -FLT_MAX;      // (finite logits further apart than float32 reaches)
        } else if (t == -1) h = m = ls = 0.0f;                      // ignored
        else { lp = h = ls = NAN; m = 0.0f; }                       // a class that does not exist
        logp[n] = lp;
        if (entropy) entropy[n] = h;
        entropy_kept[n] = h;
        top[n] = m;
        rest[n] = ls;
        classes[n] = t;
        live[n] = t == -1 ? 0 : 1;
        if (r == 0) {
            if (R == 64) bits[blockIdx.x] = word;
            else ((uint16_t*)bits)[blockIdx.x] = (uint16_t)word;
        }
    }
    if (loss) {                                                     // (given where these are all the rows)
        double sum = (double)lp;
#pragma unroll
        for (int off = R / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        if (r == 0) {
            const int c = __popcll(word);
            const double d = mean ? (double)(c > 0 ? c : 1) : 1.0;
            *loss = (float)(0.0 - sum / d);
            *each = (float)(1.0 / d);
        }
    }
}

// loss[0] = -sum logp / max(1, live rows) or -sum logp; loss[1] = what d loss / d(-logp) of a live row is
__global__ void __launch_bounds__(1024) loss_kernel(const float* __restrict__ logp, const uint8_t* __restrict__ live, int64_t rows, int mean, float* __restrict__ loss,
                                                    float* __restrict__ each) {
    __shared__ double red[16];
    __shared__ int64_t cnt[16];
    double a = 0.0;
    int64_t c = 0;
#pragma unroll 8
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
// The gradient's scale.  For one upstream value of all rows (dloss) the stored values are p - [j = t] and the factor is applied to the results.  For one per row g is stored as it
// is in float32 and bfloat16.  Float16 loses what lies below 2^-24, so there the stored values are g / table with a power of two that brings the largest possible |g| to
// 2^14, and the results are multiplied by it.
struct Upstream {
    const float* dlogp;              // per row, or null
    const float* dentropy;           // per row, or null
    const float* dloss;              // one value (with each): A_i = -dloss each for every live row
    const float* each;
    const float* table;              // scale_kernel's, or null
    int f16;
    __device__ __forceinline__ float stored() const { return dloss ? (f16 ? 16384.0f : 1.0f) : table ? table[0] : 1.0f; }
    __device__ __forceinline__ float result() const { return dloss ? *dloss * *each * (f16 ? 0x1p-14f : 1.0f) : table ? table[1] : 1.0f; }
};

// table[0]: what stored values are multiplied by, table[1]: what results are multiplied by (float16, per-row upstream values)
__global__ void __launch_bounds__(1024) scale_kernel(Upstream up, const uint8_t* __restrict__ live, int64_t rows, float* __restrict__ table) {
    __shared__ float red[16];
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
        table[0] = ldexpf(1.0f, 14 - e);
        table[1] = ldexpf(1.0f, e - 14);
    }
}

// A lane holds 4 classes of each group of 8 (register quads r4 = 0 .. 3), its partner lane ^ 32 the other 4.  Packed to 16 bits a quad is two words; exchanging the odd quad of
// the lower half with the even quad of the upper one leaves every lane with 8 neighbours - one 16-byte store: lanes < 32 those of group 2 h, the others those of group 2 h + 1.
__device__ __forceinline__ u32x4 eight_of(u32x2 even, u32x2 odd) {
    const auto a = __builtin_amdgcn_permlane32_swap(even[0], odd[0], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(even[1], odd[1], false, false);
    return u32x4{a[0], b[0], a[1], b[1]};
}
template <int DT> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT == F16) {
        typedef __attribute__((ext_vector_type(2))) _Float16 h2;
        return __builtin_bit_cast(uint32_t, h2{(_Float16)a, (_Float16)b});
    } else {
        typedef __attribute__((ext_vector_type(2))) __bf16 b2;
        return __builtin_bit_cast(uint32_t, b2{(__bf16)a, (__bf16)b});
    }
}

template <int DT> __device__ __forceinline__ float low_of(uint32_t w) {       // the value in the low 16 bits of a packed pair
    if constexpr (DT == F16) return f16_value((uint16_t)w);
    else return __builtin_bit_cast(float, w << 16);
}

// A 16-bit result tile goes to memory through the LDS, so that a wave's store covers whole rows of the tile (512 or 256 bytes) and not 32 pieces of 32 rows: 16-byte chunk c of row n
// sits at c ^ (n & 15) (& 7 in rows of 8 chunks), which keeps both the writes (32 rows, one chunk) and the reads (one row) off each other's banks.
template <class C> __device__ __forceinline__ int chunk_at(int n, int c) { return n * (2 * C::BM) + (c ^ (n & (C::BM / 8 < 16 ? C::BM / 8 - 1 : 15))) * 16; }
template <class C> __device__ __forceinline__ void put_eight(char* lds, int n, int m, const u32x4& v) {
    static_assert(C::BN * C::BM * 2 <= C::LDS_BYTES, "the tile fits");
    *(u32x4*)(lds + chunk_at<C>(n, m >> 3)) = v;
}
template <class C> __device__ __forceinline__ void flush_rows(const char* lds, uint16_t* out, int64_t stride, int rows, int cols) {
    constexpr int PER = C::BM / 8;
#pragma unroll 4
    for (int i = threadIdx.x; i < C::BN * PER; i += C::THREADS) {
        const int n = i / PER, c = i % PER;
        const u32x4 v = *(const u32x4*)(lds + chunk_at<C>(n, c));
        if (n < rows && 8 * c < cols) *(u32x4*)(out + n * stride + 8 * c) = v;
    }
}

// Sums of 32 values over the 32 lanes of each half of the wave: every exchange halves what a lane still holds (16 + 8 + 4 + 2 + 1 sums instead of 5 x 32), partners l ^ 16 (a
// row swap), then l ^ 15, l ^ 7, l ^ 2, l ^ 1.  The lane is left with the sum of value number `which`.
template <int CTRL> __device__ __forceinline__ float from_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float sums_of_32(float (&v)[32], int lane, int& which) {
    float a[16], b[8], c[4], d[2];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const auto w = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v[k]), __builtin_bit_cast(uint32_t, v[k + 16]), false, false);
        const uint32_t w0 = w[0], w1 = w[1];
        a[k] = __builtin_bit_cast(float, w0) + __builtin_bit_cast(float, w1);                   // lanes with bit 4: value k + 16
    }
    const bool b3 = lane & 8, b2 = lane & 4, b1 = lane & 2, b0 = lane & 1;
#pragma unroll
    for (int k = 0; k < 8; ++k) b[k] = (b3 ? a[k + 8] : a[k]) + from_lane<0x140>(b3 ? a[k] : a[k + 8]);
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = (b2 ? b[k + 4] : b[k]) + from_lane<0x141>(b2 ? b[k] : b[k + 4]);
#pragma unroll
    for (int k = 0; k < 2; ++k) d[k] = (b1 ? c[k + 2] : c[k]) + from_lane<0x4e>(b1 ? c[k] : c[k + 2]);
    which = lane & 31;
    return (b0 ? d[1] : d[0]) + from_lane<0xb1>(b0 ? d[0] : d[1]);
}

// a piece [c0, c1) of the classes: the logits again, and the gradient of each -> g[row][class - c0] (stride `piece`; 16 bits, float32 as three pieces g_plane values apart), zero
// up to the end of the last tile; and the sums over this tile's rows -> db_part[row tile][class]
// Bound: as statistics_kernel, and 16 bits per logit written (8192 x 2048 x 28672: 840 us, 1145 TFLOP/s, 470 MB; 50000 x 256 x 4097: 219 us in a run of passes, 268 in the first of an idle card, 416 MB).  Storing g costs less than a third
// computation of the logits, which both products would otherwise need.
// GP: pieces the gradient is stored in.  One in 16-bit types: its rounding leaves an error of the size that the result's own rounding leaves anyway (bfloat16, random upstream, 50176 rows:
// 0.0024 of the results' norm instead of 0.0017), and a second piece would double the products.  Two up to 256 rows, where the few roundings need not even out (2 rows of 2 classes: 0.004 with
// one, 0.0017 with two) and the products are bound by memory; three for float32.
template <class C, int DT, int GP, bool ENTROPY>
__global__ void __launch_bounds__(C::THREADS, C::PER_SIMD) gradient_kernel(Head hd, Upstream up, int64_t piece, int64_t g_plane, const float* __restrict__ top,
                                                              const float* __restrict__ rest, const float* __restrict__ entropy, uint16_t* __restrict__ g, float* __restrict__ db_part) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    uint32_t tm, tn, zz;
    tile_of(blockIdx.x, gridDim.x, hd.tiles_m, hd.tiles_n, tm, tn, zz);
    const int64_t m0 = hd.c0 + (int64_t)tm * C::BM, n0 = (int64_t)tn * C::BN;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave % C::WM) * (C::TM * 32), wn = (wave / C::WM) * (C::TN * 32);
    const int64_t base = m0 + wm + 4 * (lane >> 5);
    Acc<C> acc;
    struct Row { int own; float z, A, E, h; };                       // own class within the tile, -1: none, -2: the row does not count; log-sum-exp in units of log2, upstream values, entropy
    int* own_of = (int*)(lds + C::LDS_BYTES);
    float* row_of = (float*)(own_of + C::BN);
    auto row = [&](int64_t n) {
        const int64_t t = n < hd.rows ? hd.target[n] : -1;
        const bool on = t != -1;
        const float sc = up.stored();
        Row r;
        r.own = !on ? -2 : t >= m0 && t < m0 + C::BM ? (int)(t - m0) : -1;
        r.z = on ? fmaf(top[n], LOG2E, rest[n]) : 0.0f;
        r.A = on ? (up.dloss ? -1.0f : (up.dlogp ? up.dlogp[n] : 0.0f)) * sc : 0.0f;
        r.E = ENTROPY && on ? up.dentropy[n] * sc : 0.0f;
        r.h = ENTROPY && on ? entropy[n] : 0.0f;
        return r;
    };
    gemm_tile<C, DT, Elem<DT>::planes, Elem<DT>::planes, false, false>(hd.w, hd.h, m0 - hd.c0, n0, 0, hd.width, acc, lds, [&] {
        start<DT>(acc, hd.bias, base, hd.c1);
        if constexpr (C::KEEPS_ROWS)
            if (const int x = threadIdx.x; x < C::BN) {
                const Row r = row(n0 + x);
                own_of[x] = r.own; row_of[x] = r.z; row_of[C::BN + x] = r.A;
                if constexpr (ENTROPY) { row_of[2 * C::BN + x] = r.E; row_of[3 * C::BN + x] = r.h; }
            }
    });
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
        const int nl = wn + 32 * j + (lane & 31);
        Row q;
        if constexpr (C::KEEPS_ROWS) q = Row{own_of[nl], row_of[nl], row_of[C::BN + nl], ENTROPY ? row_of[2 * C::BN + nl] : 0.0f, ENTROPY ? row_of[3 * C::BN + nl] : 0.0f};
        else q = row(n0 + nl);
        const bool on = q.own != -2;
        const float z = q.z, A = q.A, El = q.E * LN2, Ah = A + q.E * q.h;
        const int rel = q.own - wm;
        const bool here = __any(rel >= 0 && rel < C::TM * 32);
        const int own = rel >= 4 * (lane >> 5) && rel < C::TM * 32 ? rel - 4 * (lane >> 5) : -1;
        float m = 0.0f, ls = 0.0f;
        auto weigh = [&](auto near) {
#pragma unroll
            for (int i = 0; i < C::TM; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float d = near ? fmaf(acc.t[i][j][r], LOG2E, -z) : fmaf(acc.t[i][j][r] - m, LOG2E, -ls), p = __builtin_amdgcn_exp2f(d);
                    acc.t[i][j][r] = ENTROPY ? -p * fmaf(El, fmaxf(d, NOTHING), Ah) : -p * A;      // g = -p (A + E (log p + H))
                }
        };
        if (__all(fabsf(z) <= NEAR * LOG2E)) weigh(std::true_type{});
        else {                                                       // one more instruction per logit
            if (on && n0 + nl < hd.rows) { m = top[n0 + nl]; ls = rest[n0 + nl]; }
            weigh(std::false_type{});
        }
        if (!__all(on))                                             // (a row that does not count is zero whatever its hidden row holds)
#pragma unroll
            for (int i = 0; i < C::TM; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc.t[i][j][r] = on ? acc.t[i][j][r] : 0.0f;
        if (here)
#pragma unroll
            for (int i = 0; i < C::TM; ++i)
                if (__any(own >= 0 && own >> 5 == i))
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc.t[i][j][r] += own == 32 * i + 8 * (r >> 2) + (r & 3) ? A : 0.0f;
    }
    if (m0 + C::BM > hd.c1) {
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (base + 32 * i + 8 * (r >> 2) + (r & 3) >= hd.c1)
#pragma unroll
                    for (int j = 0; j < C::TN; ++j) acc.t[i][j][r] = 0.0f;
    }
    if (db_part) {
        float (*red)[C::BM] = (float (*)[C::BM])lds;
#pragma unroll
        for (int i = 0; i < C::TM; i += 2) {
            float v[32];
#pragma unroll
            for (int r = 0; r < 32; ++r) {
                v[r] = i + r / 16 < C::TM ? acc.t[i + r / 16 < C::TM ? i + r / 16 : i][0][r % 16] : 0.0f;
#pragma unroll
                for (int j = 1; j < C::TN; ++j) v[r] += i + r / 16 < C::TM ? acc.t[i + r / 16 < C::TM ? i + r / 16 : i][j][r % 16] : 0.0f;
            }
            int r;
            const float sum = sums_of_32(v, lane, r);
            const int at = wm + 32 * (i + r / 16) + 8 * (r % 16 >> 2) + 4 * (lane >> 5) + (r & 3);
            if (i + r / 16 < C::TM) red[wave / C::WM][at] = sum;
        }
        __syncthreads();
        for (int m = threadIdx.x; m < C::BM; m += C::THREADS)
            if (m0 + m < hd.c1) {
                float v = red[0][m];
#pragma unroll
                for (int w = 1; w < C::WN; ++w) v += red[w][m];
                db_part[(size_t)tn * hd.classes + m0 + m] = v;
            }
        __syncthreads();
    }
    const int rows = hd.rows - n0 < C::BN ? (int)(hd.rows - n0) : C::BN;
#pragma unroll
    for (int q = 0; q < GP; ++q) {
        if (q > 0) __syncthreads();
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
            for (int i = 0; i < C::TM; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float v0 = acc.t[i][j][8 * h + 2 * r], v1 = acc.t[i][j][8 * h + 2 * r + 1];
                        w[r] = pack2<DT>(v0, v1);
                        if (q + 1 < GP) {                           // what this piece leaves for the next
                            acc.t[i][j][8 * h + 2 * r] = v0 - low_of<DT>(w[r]);
                            acc.t[i][j][8 * h + 2 * r + 1] = v1 - low_of<DT>(w[r] >> 16);
                        }
                    }
                    put_eight<C>(lds, wn + 32 * j + (lane & 31), wm + 32 * i + 16 * h + 8 * (lane >> 5), eight_of(u32x2{w[0], w[1]}, u32x2{w[2], w[3]}));
                }
        __syncthreads();
        flush_rows<C>(lds, g + q * g_plane + n0 * piece + (m0 - hd.c0), piece, rows, C::BM);
    }
}

// ------------------------------------------------------------------------------------------------------------------------------
// float32 with few rows or few classes (32 at most): memory decides, the float32 matrix instruction (16 FLOP per byte at 32) is fast enough, and laying pieces out
// would cost several times the reading: 100000 x 256 x 32 takes 59 us forward and 238 with gradients, 33 classes laid out take 107 and 377; 32 x 4096 x 4096 54 and 166, 33 rows 153 and 356.  No LDS on the way in: a lane loads 16 bytes at k = 8 q + 4 (lane >> 5) of its class, row or column and feeds them to four instructions - which
// value of k a lane holds does not matter as long as both operands hold the same.
// What lies outside is loaded from `safe` (any address that may be read) and replaced by zero, without a branch.  Loads of 16 bytes may start at any float.
typedef f32x4 __attribute__((aligned(4))) f32x4_any;
struct Skinny {
    const float *w, *h, *bias;
    int64_t w_stride, h_stride;
    int64_t rows, width, classes;
};
__device__ __forceinline__ float one_of(const float* p, const float* safe, bool in) {
    const float v = *(in ? p : safe);
    return in ? v : 0.0f;
}
__device__ __forceinline__ f32x4 four_of(const float* p, const float* safe, bool in) {          // `safe`: four values
    const f32x4 v = *(const f32x4_any*)(in ? p : safe);
    return f32x4{in ? v[0] : 0.0f, in ? v[1] : 0.0f, in ? v[2] : 0.0f, in ? v[3] : 0.0f};
}
__device__ __forceinline__ f32x4 up_to_three_of(const float* p, const float* safe, int count) {
    return f32x4{one_of(p, safe, count > 0), one_of(p + 1, safe, count > 1), one_of(p + 2, safe, count > 2), 0.0f};
}
// the logits of classes c0 .. c0 + 31 and rows r0 .. r0 + 31, a quarter of the width per wave; complete in `l` of wave 0 (register r: class c0 + 4 (lane >> 5) + 8 (r / 4) + r % 4, row r0 + lane % 32)
__device__ __forceinline__ void skinny_logits(const Skinny& q, int64_t c0, int64_t r0, float (*sums)[16][64], float (&l)[16]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, x = lane & 31, half = lane >> 5;
    const int whole = (int)(q.width & ~3), quarter = (whole + 31) / 32 * 8, k_first = wave * quarter + 4 * half, steps = quarter / 8;
    const bool w_ok = c0 + x < q.classes, h_ok = r0 + x < q.rows;
    const float *wr = w_ok ? q.w + (c0 + x) * q.w_stride : q.w, *hr = h_ok ? q.h + (r0 + x) * q.h_stride : q.h;
    f32x16 acc = {};
    auto multiply = [&](const f32x4& a, const f32x4& b) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], acc, 0, 0, 0);
    };
    constexpr int AHEAD = 8;                                                 // steps whose loads are in flight together (two sets of four in turn measured the same or slower: fewer waves fit)
    for (int s0 = 0; s0 < steps; s0 += AHEAD) {
        f32x4 a[AHEAD], b[AHEAD];
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) {
            const int k = k_first + 8 * (s0 + s);
            const bool in = s0 + s < steps && k < whole;
            a[s] = four_of(wr + k, wr, w_ok && in);
            b[s] = four_of(hr + k, hr, h_ok && in);
        }
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) multiply(a[s], b[s]);
    }
    if (wave == 3 && whole < q.width) {                                      // the last one to three values
        const int left = half == 0 ? (int)q.width - whole : 0;
        multiply(up_to_three_of(wr + whole, wr, w_ok ? left : 0), up_to_three_of(hr + whole, hr, h_ok ? left : 0));
    }
    __syncthreads();                                                         // (what was there has been read)
#pragma unroll
    for (int r = 0; r < 16; ++r) sums[wave][r][lane] = acc[r];
    __syncthreads();
    if (wave != 0) return;
    const int64_t base = c0 + 4 * (lane >> 5);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int64_t m = base + 8 * (r >> 2) + (r & 3);
        l[r] = -INFINITY;
        if (m < q.classes) {
            l[r] = (sums[0][r][lane] + sums[1][r][lane]) + (sums[2][r][lane] + sums[3][r][lane]);
            if (q.bias) l[r] += q.bias[m];
        }
    }
}

// statistics of 32 rows (workgroup / groups) over every groups-th 32 classes
template <bool ENTROPY>
__global__ void __launch_bounds__(256) skinny_statistics_kernel(Skinny q, Target target, uint32_t groups, float* __restrict__ part, float* __restrict__ own_logit) {
    __shared__ float sums[4][16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t group = blockIdx.x % groups;
    const int64_t r0 = (int64_t)(blockIdx.x / groups) * 32, n = r0 + (lane & 31), t = n < q.rows ? target.of(n) : -1;
    Stat all{-INFINITY, 0.0f, 0.0f};
    for (int64_t c0 = (int64_t)group * 32; c0 < q.classes; c0 += (int64_t)groups * 32) {
        float l[16];
        skinny_logits(q, c0, r0, sums, l);
        if (wave != 0) continue;
        const int64_t base = c0 + 4 * (lane >> 5);
        float mx = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if (t >= 0 && base + 8 * (r >> 2) + (r & 3) == t) own_logit[n] = l[r];
            mx = fmaxf(mx, l[r]);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m = mx == -INFINITY ? 0.0f : mx;
        Stat st{mx, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float d = (l[r] - m) * LOG2E, e = __builtin_amdgcn_exp2f(d);
            st.s += e;
            if constexpr (ENTROPY) st.u = fmaf(fmaxf(d, -3.0e38f), e, st.u);
        }
        st.s += __shfl_xor(st.s, 32, 64);
        if constexpr (ENTROPY) st.u += __shfl_xor(st.u, 32, 64);
        all = joined(all, st);
    }
    if (wave == 0 && lane < 32 && n < q.rows) {
        float* o = part + 3 * (size_t)group * q.rows + n;
        o[0] = all.m; o[q.rows] = all.s; o[2 * q.rows] = all.u;
    }
}

// g[row][class] in float32, rows of `stride` values (whole 32s, zero past the last class).  A workgroup takes 32 classes (workgroup % groups) and every teams-th 32 rows, and leaves the sums
// over its rows in db_part[team][class].
template <bool ENTROPY>
__global__ void __launch_bounds__(256) skinny_gradient_kernel(Skinny q, Upstream up, const int64_t* __restrict__ target, uint32_t groups, uint32_t teams, const float* __restrict__ top,
                                                              const float* __restrict__ rest, const float* __restrict__ entropy, float* __restrict__ g, int64_t stride, float* __restrict__ db_part) {
    __shared__ float sums[4][16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t team = blockIdx.x / groups;
    const int64_t c0 = (int64_t)(blockIdx.x % groups) * 32, base = c0 + 4 * (lane >> 5);
    float db[32] = {};
    for (int64_t r0 = (int64_t)team * 32; r0 < q.rows; r0 += (int64_t)teams * 32) {
        float l[16];
        skinny_logits(q, c0, r0, sums, l);
        if (wave != 0) continue;
        const int64_t n = r0 + (lane & 31), t = n < q.rows ? target[n] : -1;
        const bool on = t != -1;
        const float mrow = on ? top[n] : 0.0f, ls = on ? rest[n] : 0.0f, hrow = ENTROPY && on ? entropy[n] : 0.0f;
        const float A = on ? (up.dloss ? -1.0f : (up.dlogp ? up.dlogp[n] : 0.0f)) : 0.0f, E = ENTROPY && on ? up.dentropy[n] : 0.0f, El = E * LN2, Ah = A + E * hrow;
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            f32x4 o;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t m = base + 8 * r4 + r;
                const float d = fmaf(l[4 * r4 + r] - mrow, LOG2E, -ls), p = __builtin_amdgcn_exp2f(d);
                float v = ENTROPY ? -p * fmaf(El, fmaxf(d, NOTHING), Ah) : -p * A;
                if (m == t) v += A;
                v = on && m < q.classes ? v : 0.0f;
                o[r] = v;
                db[4 * r4 + r] += v;
            }
            if (n < q.rows) *(f32x4*)(g + n * stride + base + 8 * r4) = o;
        }
    }
    if (db_part && wave == 0) {
        int r;
        const float sum = sums_of_32(db, lane, r);                           // (values 16 .. 31 are zero)
        const int64_t m = base + 8 * (r >> 2) + (r & 3);
        if (r < 16 && m < q.classes) db_part[(size_t)team * q.classes + m] = sum;
    }
}

// dW = g^T h and dh = g W from the stored gradient, both in one launch where they take the same tiles.  The operands lie with k outermost (h, W, and g for dW): ds_read_tr turns them on the
// way from the LDS.  A sum is split over workgroups where its tiles would leave CUs idle; the parts are added in order (same bits every time), no atomics.
// Bound: the matrix pipe (8192 x 2048 x 28672, both: 1.61 - 1.66 ms, 1195 - 1160 TFLOP/s, 58 % busy; 50000 x 256 x 4097: 243 - 273 us, 865 - 770 TFLOP/s, 41 % busy: two rounds of 256 CUs).
// out[n][m] (stride out_stride): m = column of the result (width), n = its row.  slab: the sums stay in float32 [split][rows][width] for
// finish_kernel (accumulate: added to what is there); without it the scaled result is stored.
struct Product {
    Op a, b;
    int64_t k, split_k;                // length of the sum; part per split (a multiple of PART_STEP)
    int64_t rows, width;               // of the result
    uint32_t tiles_m, tiles_n;
    void* out;
    int64_t out_stride;
    int vec;                           // the result takes 16-byte stores: addresses, stride and width
    float* slab;
    int accumulate;
    const uint8_t* live;               // result rows that are zero whatever the operands hold
};

template <class C, int DT, int GP, bool AK, bool BKM>
__device__ __forceinline__ void product_tile(const Product& pr, const Upstream& up, uint32_t id, uint32_t total, char* lds) {
    typedef typename Elem<DT>::type E;
    uint32_t tm, tn, z;
    tile_of(id, total, pr.tiles_m, pr.tiles_n, tm, tn, z);
    const int64_t m0 = (int64_t)tm * C::BM, n0 = (int64_t)tn * C::BN;
    const int64_t kb = (int64_t)z * pr.split_k, ke = kb + pr.split_k < pr.k ? kb + pr.split_k : pr.k;
    Acc<C> acc;
    gemm_tile<C, DT, Elem<DT>::planes, GP, AK, BKM>(pr.a, pr.b, m0, n0, kb, ke, acc, lds, [&] { clear(acc); });
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = (wave % C::WM) * (C::TM * 32), wn = (wave / C::WM) * (C::TN * 32);
    const float sc = pr.slab ? 1.0f : up.result();
    float* slab = pr.slab ? pr.slab + (size_t)z * pr.rows * pr.width : nullptr;
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
        const int64_t n = n0 + wn + 32 * j + (lane & 31);
        const bool row = n < pr.rows, on = row && (!pr.live || pr.live[n]);
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
            const int64_t m = m0 + wm + 32 * i;
            if (pr.slab || DT == F32) {
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const int64_t mm = m + 8 * r4 + 4 * (lane >> 5);
                    float* o = pr.slab ? slab + n * pr.width + mm : (float*)pr.out + n * pr.out_stride + mm;
                    f32x4 v;
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = pr.slab ? acc.t[i][j][4 * r4 + r] : (on ? acc.t[i][j][4 * r4 + r] * sc : 0.0f);
                    if (!row) continue;
                    if (pr.vec && mm + 4 <= pr.width) {
                        if (pr.slab && pr.accumulate) v += *(const f32x4*)o;
                        *(f32x4*)o = v;
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (mm + r < pr.width) o[r] = pr.slab && pr.accumulate ? o[r] + v[r] : v[r];
                    }
                }
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = acc.t[i][j][8 * h + 2 * r] * sc, y = acc.t[i][j][8 * h + 2 * r + 1] * sc;
                        w[r] = on ? pack2<DT>(x, y) : 0u;
                    }
                    const u32x4 o8 = eight_of(u32x2{w[0], w[1]}, u32x2{w[2], w[3]});
                    const int ml = wm + 32 * i + 16 * h + 8 * (lane >> 5);
                    if (pr.vec) put_eight<C>(lds, wn + 32 * j + (lane & 31), ml, o8);
                    else if (row) {
                        E* o = (E*)pr.out + n * pr.out_stride + m0 + ml;
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            if (m0 + ml + r < pr.width) o[r] = (E)(o8[r >> 1] >> (16 * (r & 1)));
                    }
                }
            }
        }
    }
    if (DT != F32 && !pr.slab && pr.vec) {
        __syncthreads();
        flush_rows<C>(lds, (uint16_t*)pr.out + n0 * pr.out_stride + m0, pr.out_stride, pr.rows - n0 < C::BN ? (int)(pr.rows - n0) : C::BN,
                      pr.width - m0 < C::BM ? (int)(pr.width - m0) : C::BM);
    }
}

// The weights' gradient (both operands with the rows as k) and the hidden rows' (the weights with the classes as k) of one piece, in one launch: neither fills the device's last
// round alone.  groups: workgroups of the first, a multiple of 8 (the XCDs' turn) unless it is the only one.
template <class C, int DT, int GP>
__global__ void __launch_bounds__(C::THREADS, C::PER_SIMD) products_kernel(Product dw, Product dh, Upstream up, uint32_t dw_tiles, uint32_t dw_groups) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    if (blockIdx.x < dw_groups) {
        if (blockIdx.x < dw_tiles) product_tile<C, DT, GP, true, true>(dw, up, blockIdx.x, dw_tiles, lds);
    } else
        product_tile<C, DT, GP, true, false>(dh, up, blockIdx.x - dw_groups, gridDim.x - dw_groups, lds);
}
template <class C, int DT, int GP>
__global__ void __launch_bounds__(C::THREADS, C::PER_SIMD) rows_product_kernel(Product dh, Upstream up) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    product_tile<C, DT, GP, true, false>(dh, up, blockIdx.x, gridDim.x, lds);
}

// out[n][m] = sum_k a[k][m] b(k, n) for the products around a skinny gradient (m >= 4), 128 x 32 results per unit of work: b[k stride + n] (BKM) or b[n stride + k].  Lane x of a half holds columns
// m0 + 4 x .. 4 x + 3, one for each of four accumulators, so that a result's four neighbours end in one lane.  SHARED: the four waves of a workgroup take k in turns and add
// up through the LDS (long sums); else each wave has a unit of its own.
struct SkinnyProduct {
    const float *a, *b;
    int64_t a_stride, b_stride;
    const uint8_t* live;               // rows k of a that count, or null
    int64_t m, n, k, part;             // part: k per split, a multiple of 32
    uint32_t tiles_m, tiles_n, splits;
    float* out;                        // [split][n][m] slabs, or the result at out_stride
    int64_t out_stride;
    int slab;
    const uint8_t* out_live;           // result rows that are zero whatever the operands hold
};
template <bool BKM, bool SHARED>
__global__ void __launch_bounds__(256) skinny_product_kernel(SkinnyProduct q, Upstream up) {
    __shared__ float sums[SHARED ? 4 : 1][SHARED ? 64 : 1][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, x = lane & 31, half = lane >> 5;
    const uint32_t unit = SHARED ? blockIdx.x : blockIdx.x * 4 + wave;
    if (!SHARED && unit >= q.tiles_m * q.tiles_n * q.splits) return;
    const uint32_t tm = unit % q.tiles_m, tn = unit / q.tiles_m % q.tiles_n, z = unit / q.tiles_m / q.tiles_n;
    const int64_t m0 = (int64_t)tm * 128, n0 = (int64_t)tn * 32, kb = z * q.part, ke = kb + q.part < q.k ? kb + q.part : q.k;
    const bool n_ok = n0 + x < q.n;
    auto columns = [&](int i) { return m0 + 4 * i + 4 <= q.m ? m0 + 4 * i : q.m - 4; };          // of lane i; those past the last column take the last four once more
    f32x16 acc[4] = {};
    constexpr int STEP = SHARED ? 32 : 8;
    f32x4 a[2][4], b[2];                                                     // one step is loaded while the one before it is multiplied
    auto load = [&](int set, int64_t k0) {
        const int64_t k = k0 + 4 * half;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bool in = k + j < ke;
            if (q.live) in = q.live[in ? k + j : 0] != 0 && in;
            a[set][j] = four_of(q.a + (k + j) * q.a_stride + columns(x), q.a, in);
        }
        if constexpr (BKM) {
#pragma unroll
            for (int j = 0; j < 4; ++j) b[set][j] = one_of(q.b + (k + j) * q.b_stride + n0 + x, q.b, n_ok && k + j < ke);
        } else
            b[set] = four_of(q.b + (n0 + x) * q.b_stride + k, q.b, n_ok && k < ke);          // (a gradient's rows: zero from the last class to the next 32)
    };
    auto use = [&](int set) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[set][j][c], b[set][j], acc[c], 0, 0, 0);
    };
    int64_t k0 = kb + (SHARED ? 8 * wave : 0);
    load(0, k0);
    for (; k0 < ke; k0 += 2 * STEP) {
        load(1, k0 + STEP);
        use(0);
        load(0, k0 + 2 * STEP);
        use(1);
    }
    if constexpr (SHARED) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) sums[wave][16 * c + r][lane] = acc[c][r];
        __syncthreads();
    }
    if (!n_ok) return;
    float* row = q.out + (q.slab ? ((int64_t)z * q.n + n0 + x) * q.m : (n0 + x) * q.out_stride);
    const float sc = q.slab ? 1.0f : up.result();
    const bool on = q.slab || !q.out_live || q.out_live[n0 + x];
#pragma unroll
    for (int i = 0; i < (SHARED ? 4 : 16); ++i) {                            // (of four waves each finishes a quarter of the registers)
        const int r = SHARED ? 4 * wave + i : i;
        f32x4 o;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if constexpr (SHARED) o[c] = (sums[0][16 * c + r][lane] + sums[1][16 * c + r][lane]) + (sums[2][16 * c + r][lane] + sums[3][16 * c + r][lane]);
            else o[c] = acc[c][i];
            o[c] = on ? o[c] * sc : 0.0f;
        }
        *(f32x4_any*)(row + columns(8 * (r >> 2) + 4 * half + (r & 3))) = o;
    }
}

// result = scale x sum of the slabs, in their order (23 us for the slabs of 4097 x 256 and the bias at 50000 rows); and db[class] = scale x sum over the row tiles: 64 classes per workgroup, wave g takes tiles g, g + 4, ...
struct Finish {
    const float* slab;
    int64_t splits, rows, width;
    const uint8_t* live;
    void* out;
    int64_t out_stride;
    int vec;                          // width, stride and address take four values at a time
    uint32_t groups;                  // workgroups of 1024 values
};
struct FinishBias {
    const float* part;
    int64_t classes;
    int tiles;
    void* out;
    uint32_t groups;
};
template <int DT> __device__ __forceinline__ void finish(const Finish& f, float scale, uint32_t group) {
    typedef typename Elem<DT>::type E;
    const int64_t total = f.rows * f.width, i0 = ((int64_t)group * 256 + threadIdx.x) * 4;
    if (i0 >= total) return;
    if (f.vec) {
        const int64_t n = i0 / f.width, m = i0 - n * f.width;
        f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
        if (!f.live || f.live[n]) {
#pragma unroll 8
            for (int64_t s = 0; s < f.splits; ++s) a += *(const f32x4*)(f.slab + s * total + i0);
            a *= scale;
        }
        E v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = from_float<DT>(a[k]);
        __builtin_memcpy((E*)f.out + n * f.out_stride + m, v, sizeof v);
        return;
    }
    for (int64_t i = i0; i < i0 + 4 && i < total; ++i) {
        const int64_t n = i / f.width, m = i - n * f.width;
        float a = 0.0f;
        if (!f.live || f.live[n]) {
            for (int64_t s = 0; s < f.splits; ++s) a += f.slab[s * total + i];
            a *= scale;
        }
        ((E*)f.out)[n * f.out_stride + m] = from_float<DT>(a);
    }
}
template <int DT>
__global__ void __launch_bounds__(256) finish_kernel(Finish dw, Finish dh, FinishBias db, Upstream up, uint32_t from) {
    __shared__ float red[4][64];
    const float scale = up.result();
    uint32_t b = from + blockIdx.x;                                          // (from: of a launch that is not the first)
    if (b < dw.groups) return finish<DT>(dw, scale, b);
    b -= dw.groups;
    if (b < dh.groups) return finish<DT>(dh, scale, b);
    b -= dh.groups;
    const int r = threadIdx.x & 63, g = threadIdx.x >> 6;
    const int64_t j = (int64_t)b * 64 + r;
    float a = 0.0f;
    if (j < db.classes)
#pragma unroll 32
        for (int t = g; t < db.tiles; t += 4) a += db.part[(size_t)t * db.classes + j];
    red[g][r] = a;
    __syncthreads();
    if (g == 0 && j < db.classes) ((typename Elem<DT>::type*)db.out)[j] = from_float<DT>((red[0][r] + red[1][r] + red[2][r] + red[3][r]) * scale);
}

}  // namespace
}  // namespace q1head
