// learn_product.hpp -- the tiled matrix product behind the softmax loss (learn.hip): C = sum over plane pairs of A B on the matrix pipe, f32
// accumulation, with the loss's own epilogues.
//
//   SCORES  A [m x k] rows, B [n x k] rows      z = q w^T          both operands lie along k
//   DQ      A [m x k] rows, B [k x n] rows      dq = P w           B lies across k
//   DW      A [k x m] rows, B [k x n] rows      dw = P^T q         both lie across k
//
// A workgroup owns TM x TN outputs and walks k in steps of 128 bytes through a ring of two LDS stages that the load units fill by themselves
// (buffer_load ... lds, 16 bytes per lane: no register round trip).  The buffer descriptors carry the operands' true bounds, so rows, columns
// and k beyond the end arrive as zeros and no operand has to be padded.  LDS images:
//   along k:   [row][a step], 128 bytes per row, 16-byte chunks XOR-swizzled by the row (conflict-free ds_read_b128 fragments);
//   across k:  [k][columns], 32-byte units (f32: 64-byte ones) XOR-swizzled by k; the fragments of 16-bit operands come through
//              ds_read_b64_tr_b16, which hands each lane four consecutive k of one column: no transposed copy of P, the queries or the table is ever written.
// The swizzles are applied to the SOURCE address of the load (the LDS side of such a load is linear).
// The operands of the MFMA are swapped (B first): a lane then holds four consecutive COLUMNS of one output row, so row-wise softmax sums are
// mostly in-lane and stores are 8 / 16 bytes wide.
// Persistent over the output tiles: the ring runs on into the next tile while the epilogue works.
// Bound by the matrix pipe where both sides are long: 4,096 x 131,072 x 768 in bf16, scores and softmax 692 us alone (1,190 TFLOP/s; 1,344 is what a plain
// product of 8,192^3 reaches here) and 844 in a step, where the clock is lower; scores and probabilities 985, dq 866, dw 844; 300 f16 queries, whose dw is its writing, 400 TFLOP/s.  By the
// rows' reading where queries are few: one bf16 query against 10^6 rows of 768 257 us (6.0 TB/s), one f32 query against 300,000 210 us (4.4 TB/s).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "learn_device.hpp"

namespace vs {
namespace learn {

enum : int { SCORES = 0, DQ = 1, DW = 2 };
enum : int { K_F16 = 0, K_BF16 = 1, K_F32 = 2 };  // what the operands hold
enum : int { EPI_LOSS = 0, EPI_PROB = 1, EPI_PART = 2, EPI_ROWS = 3, EPI_PROB_ALONG = 4 };  // (.._ALONG: cosine, with the sums of c z per column)

struct Operand {
    const char* p;
    uint64_t plane;   // bytes between planes
    uint64_t ld;      // bytes between stored rows
    uint32_t rows;    // stored rows
    uint32_t cols;    // valid elements of a stored row (a multiple of 16 bytes)
};

struct ProductArgs {
    Operand a, b;
    uint32_t m, n, k;            // outputs and depth
    uint32_t tiles_m, tiles_n;
    uint32_t splits, ksteps;     // slices of k and steps per slice
    uint32_t segs;               // plane pairs
    uint32_t seg_a, seg_b;       // 4 bits each: the planes of pair s
    uint32_t lo_first;           // the first pair's a is the probabilities' second plane, which is stored times 2^11
    // EPI_LOSS / EPI_PROB: z2 = acc * zf * wsc * h[col] (base-2 exponent units); per row (zf, lse2, pf 2^-lo, label as bits)
    const float4* row;
    const float* h;              // nullptr: 1 (or norms)
    float* norms;                // f32: 1 / |row| of the columns is computed here, used as h and written
    const float* wsc;            // nullptr: 1
    const uint64_t* keys;        // nullptr, or per column: ~0 = not a member
    uint32_t col0;               // first column of this piece (labels are columns of the whole table, -1 = ignored)
    // EPI_LOSS
    float2* part;                // [m][part_ld] (maximum, sum of 2^(z2 - maximum)) per column tile
    uint32_t part_ld, part0;
    float2* zlab;                // z2 at the label, and what its rounding lost
    // EPI_PROB: P = f16((2^(z2 - lse2 - lo) - [label]) * pf), and 2^11 times what that loses; lo: what lse2 lost when it was rounded.  f32 operands:
    // P = (2^(z2 - lse2 - lo) - [label]) * pf * h[col] as f32; prob_kind K_BF16: the same as two bf16
    int prob_kind;
    const float* lo;
    uint16_t* prob;
    uint64_t prob_plane;         // elements
    uint32_t prob_ld, prob_planes;
    float* tpart;                // EPI_PROB_ALONG: [wave rows of tiles][n]: sums over rows of dloss c z
    const float* graw;           // dloss per row
    // EPI_PART
    float* out_part;             // [splits][m][n]
    // EPI_ROWS
    void* out;
    int out_scalar;
    uint64_t out_ld;             // elements
    const float* wf;             // nullptr: 1
    const float* rf;             // nullptr: 1; per output row
    const float* tcoef;          // nullptr, or per output row: minus tcoef * (tinv * raw row)
    const float* tinv;
    const void* raw;
    int raw_scalar;
    uint64_t raw_ld;
};

// A step is 128 bytes of k: 64 16-bit elements, 32 f32.
template <int KIND>
constexpr uint32_t kES = KIND == K_F32 ? 4u : 2u;
template <int KIND>
constexpr uint32_t kBK = 128u / kES<KIND>;

__device__ __forceinline__ uint32_t swz_row(uint32_t row) { return (row >> 1) & 7u; }
template <int COLS>
__device__ __forceinline__ uint32_t swz_k(uint32_t k) {
    return ((k & 3u) | (((k >> 3) & 1u) << 2)) & (COLS / 16 - 1u);
}

// One operand's stages: 64 deep, X output rows / columns wide (X * 128 bytes of LDS), brought in by NW waves in pieces of 1 KiB.  Between
// two steps only a scalar moves; the instructions between a step's barrier and its first MFMA are what every wave of the CU waits for
// (a descriptor computed per step cost 190 of 800 us at 4,096 x 131,072 x 768).
template <int X, int NW, bool ACROSS, int KIND>
struct Loader {
    static constexpr uint32_t ES = kES<KIND>, BK = kBK<KIND>;
    static constexpr int PIECES = X / 8 / NW;
    static_assert(X % (8 * NW) == 0, "whole pieces per wave");
    uint32_t off[PIECES];
    const char* base;       // of the tile's first row / column (along), of the step (across)
    uint32_t limit, full;   // bytes behind base that belong to the operand; across: of a step 64 deep
    __device__ __forceinline__ void init(uint64_t ld, uint32_t w, uint32_t lane) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const uint32_t at = (w * PIECES + i) * 1024u + lane * 16u;
            if constexpr (ACROSS) {
                const uint32_t kr = at / (X * ES), cp = (at % (X * ES)) >> 4;
                const uint32_t c = KIND == K_F32 ? cp ^ (((kr >> 2) & 3u) << 2) : cp ^ (swz_k<X>(kr) << 1);
                off[i] = kr * (uint32_t)ld + c * 16u;
            } else {
                const uint32_t row = at >> 7, cp = (at >> 4) & 7u;
                off[i] = row * (uint32_t)ld + ((cp ^ swz_row(row)) << 4);
            }
        }
    }
    static __device__ __forceinline__ uint32_t clamped(uint64_t bytes) { return bytes > 0x7FFFF000ull ? 0x7FFFF000u : (uint32_t)bytes; }
    // x0: first output row / column of the tile; k0: first k of the step; kend: end of k
    __device__ __forceinline__ void open(const Operand& o, uint32_t plane, uint32_t x0, uint32_t k0, uint32_t kend) {
        if constexpr (ACROSS) {
            base = o.p + plane * o.plane + (uint64_t)k0 * o.ld + (uint64_t)x0 * ES;
            full = x0 < o.cols ? clamped((BK - 1u) * o.ld + (uint64_t)(o.cols - x0) * ES) : 0u;
            depth(o, k0, kend);
        } else {
            base = o.p + plane * o.plane + (uint64_t)x0 * o.ld;
            limit = x0 < o.rows ? clamped((uint64_t)(o.rows - x0) * o.ld) : 0u;
        }
    }
    __device__ __forceinline__ void depth(const Operand& o, uint32_t k0, uint32_t kend) {
        const uint32_t left = k0 < kend ? kend - k0 : 0u;
        const uint32_t less = left < BK ? (BK - left) * (uint32_t)o.ld : 0u;
        limit = left && less < full ? full - less : 0u;
    }
    __device__ __forceinline__ void advance(const Operand& o, uint32_t k0, uint32_t kend) {  // to the next step, at k0
        if constexpr (ACROSS) {
            base += (uint64_t)BK * o.ld;
            depth(o, k0, kend);
        }
    }
    __device__ __forceinline__ void piece(int i, bool more, uint32_t k0, uint32_t kend, char* lds, uint32_t w, uint32_t lane) const {
        // (all of it the same in every lane: kept in scalar registers, or each load becomes a loop over the lanes' descriptors)
        const uint32_t bytes = __builtin_amdgcn_readfirstlane(more ? limit : 0u), lo = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)base),
                       hi = __builtin_amdgcn_readfirstlane((uint32_t)((uintptr_t)base >> 32));
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)((uintptr_t)hi << 32 | lo), 0, (int)bytes, 0x00020000);
        const bool tail = !ACROSS && k0 + BK > kend;  // the last step of a depth that is no multiple of a step: chunks beyond it read nothing
        const uint32_t shift = ACROSS || tail ? 0u : k0 * ES;
        uint32_t v = off[i];
        if (tail) {
            const uint32_t row = (w * PIECES + i) * 8u + (lane >> 3);
            const uint32_t kc = ((lane & 7u) ^ swz_row(row)) * (16u / ES);
            v = k0 + kc < kend ? v + k0 * ES : 0x7FFFFFF0u;
        }
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds + (w * PIECES + i) * 1024u), 16, v, shift, 0, 0);
    }
};

__device__ __forceinline__ void stage_rows(const void* p, uint32_t bytes, uint32_t off, char* lds) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)bytes, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, off, 0, 0, 0);
}

// Fragment of 16 output rows / columns x 32 k (eight k per lane: k = kk * 32 + 8 * (lane / 16) + 0..7), operand along k.
template <class Frag>
__device__ __forceinline__ Frag read_fragment(const char* lds, uint32_t x, uint32_t kk, uint32_t lane) {
    const uint32_t row = x + (lane & 15u), kc = kk * 4u + (lane >> 4);
    return *reinterpret_cast<const Frag*>(lds + row * 128u + ((kc ^ swz_row(row)) << 4));
}
// The same, operand across k: two transposing reads per fragment.  Lane i of 16 names 8 bytes of k row (i / 4), columns 4 * (i % 4), and gets
// column i of four k.  swz_k is the same for every kk and for both halves of a fragment, so one address per fragment and immediate offsets do.
// Written out, with their wait in the same block: behind the builtin the compiler waits for the LDS loads in flight (the next stage's).
template <int X>
__device__ __forceinline__ uint32_t across_address(uint32_t x, uint32_t lane) {
    const uint32_t i = lane & 15u, k = (lane >> 4) * 8u + (i >> 2);
    return k * (X * 2u) + (((x >> 4) ^ swz_k<X>(k)) << 5) + (i & 3u) * 8u;
}
using s16x4 = __attribute__((ext_vector_type(4))) short;
using s16x8 = __attribute__((ext_vector_type(8))) short;
template <int X, int KK>
__device__ __forceinline__ void read_across4(const uint32_t* a, s16x8* f) {
    s16x4 l0, h0, l1, h1, l2, h2, l3, h3;
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
        "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
        "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
        "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(l0), "=&v"(h0), "=&v"(l1), "=&v"(h1), "=&v"(l2), "=&v"(h2), "=&v"(l3), "=&v"(h3)
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(KK * 64 * X), "n"(KK * 64 * X + 8 * X)
        : "memory");
    f[0] = __builtin_shufflevector(l0, h0, 0, 1, 2, 3, 4, 5, 6, 7);
    f[1] = __builtin_shufflevector(l1, h1, 0, 1, 2, 3, 4, 5, 6, 7);
    f[2] = __builtin_shufflevector(l2, h2, 0, 1, 2, 3, 4, 5, 6, 7);
    f[3] = __builtin_shufflevector(l3, h3, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <int X, int KK>
__device__ __forceinline__ void read_across2(const uint32_t* a, s16x8* f) {
    s16x4 l0, h0, l1, h1;
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
        "ds_read_b64_tr_b16 %2, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(l0), "=&v"(h0), "=&v"(l1), "=&v"(h1)
        : "v"(a[0]), "v"(a[1]), "n"(KK * 64 * X), "n"(KK * 64 * X + 8 * X)
        : "memory");
    f[0] = __builtin_shufflevector(l0, h0, 0, 1, 2, 3, 4, 5, 6, 7);
    f[1] = __builtin_shufflevector(l1, h1, 0, 1, 2, 3, 4, 5, 6, 7);
}
// T fragments of one operand; at: LDS byte address of its stage.  f32: a lane's four elements are those of four MFMAs, k = kk * 16 +
// 4 * (lane / 16) + 0..3 (which k an MFMA multiplies does not matter as long as both operands agree).
template <int X, int T, bool ACROSS, int KIND, int KK, class Frag>
__device__ __forceinline__ void read_fragments(const char* lds, uint32_t at, uint32_t x, uint32_t lane, const uint32_t* addr, Frag* f) {
    if constexpr (ACROSS && KIND == K_F32) {
        const uint32_t g = lane >> 4;
#pragma unroll
        for (int i = 0; i < T; ++i) {
            const uint32_t col = ((x + i * 16u + (lane & 15u)) * 4u) ^ (g << 6);
#pragma unroll
            for (int t = 0; t < 4; ++t) f[i][t] = *reinterpret_cast<const float*>(lds + (KK * 16u + g * 4u + t) * (X * 4u) + col);
        }
    } else if constexpr (ACROSS) {
        uint32_t a[T];
        s16x8 v[T];
#pragma unroll
        for (int i = 0; i < T; ++i) a[i] = addr[i] + at;
        if constexpr (T == 8) {
            read_across4<X, KK>(a, v);
            read_across4<X, KK>(a + 4, v + 4);
        } else if constexpr (T == 4) {
            read_across4<X, KK>(a, v);
        } else {
            static_assert(T == 2, "fragments per wave");
            read_across2<X, KK>(a, v);
        }
#pragma unroll
        for (int i = 0; i < T; ++i) f[i] = __builtin_bit_cast(Frag, v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < T; ++i) f[i] = read_fragment<Frag>(lds, x + i * 16u, KK, lane);
    }
}

// MFMAS: how many a fragment feeds
template <int KIND>
struct Matrix {
    static constexpr int MFMAS = 1;
    using frag = __attribute__((ext_vector_type(8))) _Float16;
    static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c, int) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Matrix<K_BF16> {
    static constexpr int MFMAS = 1;
    using frag = __attribute__((ext_vector_type(8))) __bf16;
    static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c, int) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Matrix<K_F32> {
    static constexpr int MFMAS = 4;
    using frag = f32x4;
    static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c, int t) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a[t], b[t], c, 0, 0, 0); }
};

// 16 rows x 64 columns of 16-bit values, four consecutive columns of a row per lane and block, to memory as whole 128-byte lines: straight
// from the registers a store instruction would touch 16 rows in 32-byte pieces (measured: 850 us for 268 MB of probabilities; so 255 us).
// cols (a multiple of 8) bounds the columns; 16-byte aligned rows.  scratch: the wave's own, for ROWS rows at a time.
template <int ROWS>
__device__ __forceinline__ void store_lines(char* scratch, const ushort4 (&v)[4], uint16_t* to, uint64_t ld, uint32_t row, uint32_t rows, uint32_t col, uint32_t cols,
                                            uint32_t lane) {
    const uint32_t r = lane & 15u, q = lane >> 4;
#pragma unroll
    for (uint32_t part = 0; part < 16u / ROWS; ++part) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the last block has been read)
        if (ROWS == 16 || r / ROWS == part) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                *reinterpret_cast<ushort4*>(scratch + (r % ROWS) * 128u + (((j * 2u + (q >> 1)) ^ (r & 7u)) << 4) + (q & 1u) * 8u) = v[j];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (uint32_t h = 0; h < ROWS / 8; ++h) {
            const uint32_t in = h * 8u + (lane >> 3), rr = part * ROWS + in, c = lane & 7u;
            const uint4 x = *reinterpret_cast<const uint4*>(scratch + in * 128u + ((c ^ (in & 7u)) << 4));
            if (row + rr < rows && col + c * 8u < cols) *reinterpret_cast<uint4*>(to + (uint64_t)(row + rr) * ld + col + c * 8u) = x;
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// 16 rows x 64 columns of f32 alike, 32 columns at a time.  less: what is subtracted on the way (load_lines of a table) times ti times tc, the row's
// (lane & 15) factors (in this order: 1 / |row|^2 may not exist in f32; tc 0: nothing is).
__device__ __forceinline__ void load_lines(const float* from, uint64_t ld, uint32_t row, uint32_t rows, uint32_t col, uint32_t cols, uint32_t lane, f32x4 (&v)[4]) {
#pragma unroll
    for (uint32_t x = 0; x < 4; ++x) {
        const uint32_t rr = (x & 1u) * 8u + (lane >> 3), at = col + (x >> 1) * 32u + (lane & 7u) * 4u;
        v[x] = row + rr < rows && at < cols ? *reinterpret_cast<const f32x4*>(from + (uint64_t)(row + rr) * ld + at) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
}
template <int ROWS>
__device__ __forceinline__ void store_lines(char* scratch, const f32x4 (&v)[4], float* to, uint64_t ld, uint32_t row, uint32_t rows, uint32_t col, uint32_t cols,
                                            uint32_t lane, const f32x4* less = nullptr, float tc = 0.f, float ti = 0.f) {
    const uint32_t r = lane & 15u, q = lane >> 4, c = lane & 7u;
#pragma unroll
    for (uint32_t half = 0; half < 2; ++half)
#pragma unroll
        for (uint32_t part = 0; part < 16u / ROWS; ++part) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the last block has been read)
            if (ROWS == 16 || r / ROWS == part) {
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j) *reinterpret_cast<f32x4*>(scratch + (r % ROWS) * 128u + (((j * 4u + q) ^ (r & 7u)) << 4)) = v[half * 2u + j];
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (uint32_t h = 0; h < ROWS / 8; ++h) {
                const uint32_t in = h * 8u + (lane >> 3), rr = part * ROWS + in, at = col + half * 32u + c * 4u;
                f32x4 x = *reinterpret_cast<const f32x4*>(scratch + in * 128u + ((c ^ (in & 7u)) << 4));
                if (less) {
                    const float t = __shfl(tc, rr), i = __shfl(ti, rr);
                    if (t != 0.f) x -= less[half * 2u + part * ROWS / 8u + h] * i * t;
                }
                if (row + rr < rows && at < cols) *reinterpret_cast<f32x4*>(to + (uint64_t)(row + rr) * ld + at) = x;
            }
            __builtin_amdgcn_wave_barrier();
        }
}

// WM x WN waves, each MT x NT blocks of 16 x 16.
template <int TM_, int TN_, int WM_, int WN_, int RING_>
struct Shape {
    static constexpr int RING = RING_;  // stages in LDS: the loads run RING - 1 steps ahead
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, NW = WM_ * WN_;
    static constexpr int MT = TM_ / WM_ / 16, NT = TN_ / WN_ / 16;
    static constexpr int A_BYTES = TM_ * 128, B_BYTES = TN_ * 128, STAGE = A_BYTES + B_BYTES;
    // row factors of RING tiles, then EPI_LOSS: (maximum, sum) per wave column and row; else SCRATCH per wave
    static constexpr int ROW_BYTES = TM_ * 16 < 1024 ? 1024 : TM_ * 16;  // (a wave brings 1024 at a time)
    static constexpr int SCRATCH = RING_ * (STAGE + ROW_BYTES) + NW * 2048 <= 160 * 1024 ? 2048 : 1024;  // of a wave: 16 or 8 rows of 128 bytes
    static constexpr int EPI_BYTES = RING_ * ROW_BYTES + (WN_ * TM_ * 8 > NW * SCRATCH ? WN_ * TM_ * 8 : NW * SCRATCH);
    static constexpr int LDS = RING_ * STAGE + EPI_BYTES;
};
using Large = Shape<256, 256, 2, 4, 2>;   // one workgroup per CU, 152 KiB of LDS
using Medium = Shape<128, 256, 2, 4, 3>;  // one workgroup per CU, 158 KiB
using Small = Shape<64, 128, 2, 2, 2>;    // 58 KiB: two workgroups per CU
using Slim = Shape<32, 128, 1, 2, 2>;     // 46 KiB: three workgroups per CU, for up to 32 f32 queries (their padding to 64 is the small tile's time)

template <class S, int FORM, int EPI, int KIND>
__global__ __launch_bounds__(S::NW * 64) void product_kernel(ProductArgs g) {
    constexpr bool A_ACROSS = FORM == DW, B_ACROSS = FORM != SCORES;
    constexpr bool SOFTMAX = FORM == SCORES;
    constexpr uint32_t BK = kBK<KIND>;
    constexpr int SCRATCH = S::SCRATCH;
    using H = Matrix<KIND>;
    using frag = typename H::frag;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const uint32_t lane = threadIdx.x & 63u, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = w / S::WN, wn = w % S::WN;
    // Blocks b, b + 8, b + 16 ... share an XCD and its L2: each XCD takes a contiguous share of the tiles, ordered so that the tiles in
    // flight on its 32 CUs are a compact patch (8 row tiles by 4 column tiles of the scores; all column tiles of a row tile of the gradients):
    // an operand's stage is fetched once per XCD and read by the others from L2.
    constexpr uint32_t GROUP = FORM == SCORES ? 4u : 8u;
    const uint32_t per_split = g.tiles_m * g.tiles_n, all = per_split * g.splits;
    const uint32_t share = (all + 7u) / 8u, first = (blockIdx.x & 7u) * share;
    const uint32_t mine = first < all ? (all - first < share ? all - first : share) : 0u;  // tiles of this XCD
    const uint32_t step = gridDim.x >> 3;                                                  // (the grid: a multiple of 8)
    const uint32_t tile0 = blockIdx.x >> 3;
    if (tile0 >= mine) return;
    const auto place = [&](uint32_t t, uint32_t& tm, uint32_t& tn, uint32_t& sp) {
        t += first;
        sp = t / per_split;
        const uint32_t r = t - sp * per_split;
        const uint32_t group = r / (GROUP * g.tiles_m), in = r - group * GROUP * g.tiles_m;
        const uint32_t left = g.tiles_n - group * GROUP, width = left < GROUP ? left : GROUP;
        tm = in / width;
        tn = group * GROUP + in % width;
    };
    Loader<S::TM, S::NW, A_ACROSS, KIND> la;
    Loader<S::TN, S::NW, B_ACROSS, KIND> lb;
    la.init(g.a.ld, w, lane);
    lb.init(g.b.ld, w, lane);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    uint32_t aa[S::MT], ab[S::NT];  // (across) the fragments' addresses within a stage
#pragma unroll
    for (int i = 0; i < S::MT; ++i) aa[i] = A_ACROSS ? across_address<S::TM>((wm * S::MT + i) * 16u, lane) : 0u;
#pragma unroll
    for (int j = 0; j < S::NT; ++j) ab[j] = B_ACROSS ? across_address<S::TN>((wn * S::NT + j) * 16u, lane) : 0u;
    const uint32_t steps = g.ksteps * g.segs;
    const uint32_t total = ((mine - 1u - tile0) / step + 1u) * steps;
    char* const row_buffers = lds + S::RING * S::STAGE;  // SOFTMAX: the row factors of RING tiles (a tile may be one step)
    uint32_t p = 0, p_tile = tile0, p_seg = 0, p_ks = 0, p_tm, p_tn, p_sp, p_k0, p_parity = 0;
    const auto open = [&]() {
        p_k0 = p_sp * g.ksteps * BK;
        la.open(g.a, (g.seg_a >> (4u * p_seg)) & 15u, p_tm * S::TM, p_k0, g.k);
        lb.open(g.b, (g.seg_b >> (4u * p_seg)) & 15u, p_tn * S::TN, p_k0, g.k);
    };
    const auto prefetch_rows = [&]() {
        // (beyond the last step the operands have no bytes: the loads bring zeros nobody reads)
        if (SOFTMAX) {
            if (p < total && p_ks == 0 && p_seg == 0 && w < (S::TM + 63u) / 64u) {  // (rows beyond the last: zeros)
                const uint32_t r0 = p_tm * S::TM;
                stage_rows(g.row + r0, (g.m - r0) * 16u, w * 1024u + lane * 16u, row_buffers + p_parity * S::ROW_BYTES + w * 1024u);
            }
        }
    };
    const auto advance = [&]() {
        ++p;
        if (++p_ks < g.ksteps) {
            p_k0 += BK;
            la.advance(g.a, p_k0, g.k);
            lb.advance(g.b, p_k0, g.k);
            return;
        }
        p_ks = 0;
        if (++p_seg == g.segs) {
            p_seg = 0;
            p_parity = p_parity + 1u < (uint32_t)S::RING ? p_parity + 1u : 0u;
            p_tile += step;
            if (p_tile < mine) place(p_tile, p_tm, p_tn, p_sp);  // (beyond the last tile: the last one's operands, of no bytes)
        }
        open();
    };
    constexpr int PA = decltype(la)::PIECES, P = PA + decltype(lb)::PIECES;
    place(p_tile, p_tm, p_tn, p_sp);
    open();
    prefetch_rows();
    uint32_t next_at = 0;  // of the stage the next loads go to
#pragma unroll
    for (int st = 0; st < S::RING - 1; ++st) {
        if (st) prefetch_rows();
#pragma unroll
        for (int x = 0; x < P; ++x) {
            if (x < PA) la.piece(x, p < total, p_k0, g.k, lds + next_at, w, lane);
            else lb.piece(x - PA, p < total, p_k0, g.k, lds + next_at + S::A_BYTES, w, lane);
        }
        advance();
        next_at += S::STAGE;
    }
    const float wsc = SOFTMAX && g.wsc ? *g.wsc : 1.f;
    uint32_t stage = 0, parity = 0;
    for (uint32_t tile = tile0; tile < mine; tile += step, parity = parity + 1u < (uint32_t)S::RING ? parity + 1u : 0u) {
        uint32_t tm, tn, sp;
        place(tile, tm, tn, sp);
        // (f32 scores in two sums, added at the end: half of the terms and of the size each, so less rounding; four leave one wave per SIMD)
        constexpr int SUMS = SOFTMAX && KIND == K_F32 ? 2 : 1;
        f32x4 acc[S::MT][S::NT], more[SUMS][S::MT][S::NT];
#pragma unroll
        for (int i = 0; i < S::MT; ++i)
#pragma unroll
            for (int j = 0; j < S::NT; ++j) {
                acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int t = 1; t < SUMS; ++t) more[t][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        // f32 rows under a cosine bring their lengths with them: a column's elements lie in the four lanes of its number
        const bool own = SOFTMAX && KIND == K_F32 && g.norms;
        float ss[S::NT];
#pragma unroll
        for (int j = 0; j < S::NT; ++j) ss[j] = 0.f;
        for (uint32_t s = 0; s < steps; ++s) {
            // (a wave's loads arrive in order: what may still be on its way are the P pieces of the stages after this one)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S::RING - 2) * P) : "memory");
            __builtin_amdgcn_s_barrier();  // the stage is whole; nobody reads the one before it any more
            asm volatile("" ::: "memory");
            prefetch_rows();
            if constexpr (FORM != SCORES) {
                if (KIND == K_F16 && g.lo_first && s == g.ksteps) {
#pragma unroll
                    for (int i = 0; i < S::MT; ++i)
#pragma unroll
                        for (int j = 0; j < S::NT; ++j) acc[i][j] *= 0x1p-11f;
                }
            }
            const char* sa = lds + stage;
            const char* sb = sa + S::A_BYTES;
            char* next = lds + next_at;
            // The next stage's loads go out one by one between the MFMAs of the step's first half: issued in a row they fill the queue of the
            // load unit (16 cycles each, 64 of them per CU), and every wave stands in front of its first MFMA until its own are through.
            frag fa[S::MT], fb[S::NT];
            const auto square = [&]() {
                if constexpr (SOFTMAX && KIND == K_F32) {
                    if (!own) return;
#pragma unroll
                    for (int j = 0; j < S::NT; ++j)
#pragma unroll
                        for (int t = 0; t < 4; ++t) ss[j] = fmaf(fb[j][t], fb[j][t], ss[j]);
                }
            };
            read_fragments<S::TM, S::MT, A_ACROSS, KIND, 0>(sa, lds0 + stage, wm * S::MT * 16u, lane, aa, fa);
            read_fragments<S::TN, S::NT, B_ACROSS, KIND, 0>(sb, lds0 + stage + S::A_BYTES, wn * S::NT * 16u, lane, ab, fb);
#pragma unroll
            for (int i = 0; i < S::MT; ++i) {
#pragma unroll
                for (int j = 0; j < S::NT; ++j) acc[i][j] = H::mma(fb[j], fa[i], acc[i][j], 0);
                __builtin_amdgcn_sched_barrier(0x104);  // (scalar instructions and LDS reads may pass)
#pragma unroll
                for (int x = i * P / S::MT; x < (i + 1) * P / S::MT; ++x) {
                    if (x < PA) la.piece(x, p < total, p_k0, g.k, next, w, lane);
                    else lb.piece(x - PA, p < total, p_k0, g.k, next + S::A_BYTES, w, lane);
                }
                __builtin_amdgcn_sched_barrier(0x104);
            }
#pragma unroll
            for (int t = 1; t < H::MFMAS; ++t)
#pragma unroll
                for (int i = 0; i < S::MT; ++i)
#pragma unroll
                    for (int j = 0; j < S::NT; ++j) {
                        f32x4& c = t % SUMS ? more[t % SUMS][i][j] : acc[i][j];
                        c = H::mma(fb[j], fa[i], c, t);
                    }
            square();
            read_fragments<S::TM, S::MT, A_ACROSS, KIND, 1>(sa, lds0 + stage, wm * S::MT * 16u, lane, aa, fa);
            read_fragments<S::TN, S::NT, B_ACROSS, KIND, 1>(sb, lds0 + stage + S::A_BYTES, wn * S::NT * 16u, lane, ab, fb);
#pragma unroll
            for (int t = 0; t < H::MFMAS; ++t)
#pragma unroll
                for (int i = 0; i < S::MT; ++i)
#pragma unroll
                    for (int j = 0; j < S::NT; ++j) {
                        f32x4& c = t % SUMS ? more[t % SUMS][i][j] : acc[i][j];
                        c = H::mma(fb[j], fa[i], c, t);
                    }
            square();
            advance();
            next_at = stage;
            stage = stage + S::STAGE < S::RING * S::STAGE ? stage + S::STAGE : 0u;
        }
#pragma unroll
        for (int t = 1; t < SUMS; ++t)
#pragma unroll
            for (int i = 0; i < S::MT; ++i)
#pragma unroll
                for (int j = 0; j < S::NT; ++j) acc[i][j] += more[t][i][j];
        // lane: row (lane & 15) of a 16 x 16 block, columns 4 * (lane / 16) + 0..3
        const uint32_t row0 = tm * S::TM + wm * S::MT * 16u + (lane & 15u);
        const uint32_t c0 = tn * S::TN + wn * S::NT * 16u, cl = c0 + (lane >> 4) * 4u;
        char* scratch = lds + S::RING * (S::STAGE + S::ROW_BYTES) + w * (uint32_t)SCRATCH;
        if constexpr (SOFTMAX) {
            const float4* rows = reinterpret_cast<const float4*>(row_buffers + parity * S::ROW_BYTES);
            // columns that all exist: the common case, with fewer instructions per score (the epilogue's vector instructions are what a product of
            // short rows waits for: 128 scores per lane)
            const bool plain = !g.keys && c0 + S::NT * 16u <= g.n;
            f32x4 h[S::NT];
            uint32_t live[S::NT];  // bit r: column j, r exists
            const bool scaled = own || g.h;
            if (own) {
#pragma unroll
                for (int j = 0; j < S::NT; ++j) {
                    ss[j] += __shfl_xor(ss[j], 16);
                    ss[j] += __shfl_xor(ss[j], 32);
                    const float inv = ss[j] > 0.f ? 1.f / sqrtf(ss[j]) : 0.f;
                    const uint32_t c = c0 + j * 16u + lane;
                    if (tm == 0 && wm == 0 && lane < 16u && c < g.n) g.norms[c] = inv;
#pragma unroll
                    for (int r = 0; r < 4; ++r) h[j][r] = __shfl(inv, (lane >> 4) * 4u + r);
                }
            }
            if (!plain) {
#pragma unroll
                for (int j = 0; j < S::NT; ++j) {
                    live[j] = 0;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint32_t c = cl + j * 16u + r;
                        const bool in = c < g.n && !(g.keys && g.keys[c] == ~0ull);
                        live[j] |= in ? 1u << r : 0u;
                        h[j][r] = !in ? 0.f : own ? h[j][r] : g.h ? g.h[c] : 1.f;
                    }
                }
            } else if (g.h) {  // (own: they are there)
#pragma unroll
                for (int j = 0; j < S::NT; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) h[j][r] = g.h[cl + j * 16u + r];
            }
            if (scaled) {
#pragma unroll
                for (int i = 0; i < S::MT; ++i)
#pragma unroll
                    for (int j = 0; j < S::NT; ++j) acc[i][j] *= h[j];
            }
            if constexpr (EPI == EPI_LOSS) {
                float2* red = reinterpret_cast<float2*>(lds + S::RING * (S::STAGE + S::ROW_BYTES));
                float2 ms[S::MT];  // of this lane's 16 columns
#pragma unroll
                for (int i = 0; i < S::MT; ++i) {
                    const float4 rf = rows[(wm * S::MT + i) * 16u + (lane & 15u)];
                    const float f = rf.x * wsc;
                    const uint32_t lab = (uint32_t)(__float_as_int(rf.w) - (int32_t)g.col0) - cl;
                    const bool here = __any(lab < S::NT * 16u);  // a label of these rows lies in the wave's columns
                    // the sum leaves the label out: the loss is log(1 + the others' share), which keeps its accuracy when it is small.
                    // 2^(acc f - top) in one rounding: what the score itself loses when it is rounded does not enter.
                    float top = -__builtin_inff(), sum = 0.f;
                    if (plain && !here) {
                        float most = acc[i][0][0], least = most;
#pragma unroll
                        for (int j = 0; j < S::NT; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) most = fmaxf(most, acc[i][j][r]), least = fminf(least, acc[i][j][r]);
                        top = (f >= 0.f ? most : least) * f;
                        const float base = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
                        for (int j = 0; j < S::NT; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) sum += exp2_fast(fmaf(acc[i][j][r], f, -base));
                    } else {
#pragma unroll
                        for (int j = 0; j < S::NT; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float z = acc[i][j][r] * f;
                                bool in = plain || ((live[j] >> r) & 1u);
                                if (lab == j * 16u + r) {
                                    if (row0 + i * 16u < g.m) g.zlab[row0 + i * 16u] = make_float2(z, fabsf(z) < __builtin_inff() ? fmaf(acc[i][j][r], f, -z) : 0.f);
                                    in = false;
                                }
                                top = in ? fmaxf(top, z) : top;
                            }
                        const float base = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
                        for (int j = 0; j < S::NT; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float e = exp2_fast(fmaf(acc[i][j][r], f, -base));
                                sum += (plain || ((live[j] >> r) & 1u)) && lab != j * 16u + r ? e : 0.f;
                            }
                    }
                    ms[i] = make_float2(top, sum);
                }
                // the four lanes of a row: block pairs swap halves, so that a join serves two blocks of rows at once
                if constexpr (S::MT == 8) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) ms[i] = join_swapped<32>(ms[2 * i], ms[2 * i + 1]);
                    ms[0] = join_swapped<16>(ms[0], ms[1]);
                    ms[1] = join_swapped<16>(ms[2], ms[3]);
                    const uint32_t q = lane >> 4, i = (q & 1u) * 2u + (q >> 1);
                    red[wn * S::TM + (wm * S::MT + i) * 16u + (lane & 15u)] = ms[0];
                    red[wn * S::TM + (wm * S::MT + 4u + i) * 16u + (lane & 15u)] = ms[1];
                } else if constexpr (S::MT == 4) {
                    ms[0] = join_swapped<32>(ms[0], ms[1]);
                    ms[1] = join_swapped<32>(ms[2], ms[3]);
                    ms[0] = join_swapped<16>(ms[0], ms[1]);
                    const uint32_t q = lane >> 4, i = (q & 1u) * 2u + (q >> 1);
                    red[wn * S::TM + (wm * S::MT + i) * 16u + (lane & 15u)] = ms[0];
                } else {
                    static_assert(S::MT == 2, "row blocks per wave");
                    float2 a = join_swapped<32>(ms[0], ms[1]);
                    a = join_sums(a, make_float2(__shfl_xor(a.x, 16), __shfl_xor(a.y, 16)));
                    if (!(lane & 16u)) red[wn * S::TM + (wm * S::MT + (lane >> 5)) * 16u + (lane & 15u)] = a;
                }
                __syncthreads();
                for (uint32_t t = threadIdx.x; t < (uint32_t)S::TM; t += S::NW * 64) {
                    const uint32_t row = tm * S::TM + t;
                    if (row < g.m) {
                        float2 a = red[t];
#pragma unroll
                        for (int x = 1; x < S::WN; ++x) a = join_sums(a, red[x * S::TM + t]);
                        g.part[(size_t)row * g.part_ld + g.part0 + tn] = a;
                    }
                }
                // (the next tile's writes here come after its first step's barrier: these reads are done by then)
            } else {
                if constexpr (EPI == EPI_PROB_ALONG) {
                    // (a pass of its own, four columns at a time: its sums and the probabilities' stores together do not fit the registers)
                    float gr[S::MT], lo[S::MT];
#pragma unroll
                    for (int i = 0; i < S::MT; ++i) {
                        const bool has = row0 + i * 16u < g.m;
                        gr[i] = has ? g.graw[row0 + i * 16u] : 0.f;
                        lo[i] = has ? g.lo[row0 + i * 16u] : 0.f;
                    }
#pragma unroll
                    for (int j = 0; j < S::NT; ++j) {
                        f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int i = 0; i < S::MT; ++i) {
                            const float4 rf = rows[(wm * S::MT + i) * 16u + (lane & 15u)];
                            const uint32_t lab = (uint32_t)(__float_as_int(rf.w) - (int32_t)g.col0) - cl - j * 16u;
                            float f = rf.x * wsc;
                            asm volatile("" : "+v"(f));  // (or the compiler keeps all 128 probabilities for the next pass)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float z = acc[i][j][r] * f;
                                const float q = exp2_fast(fmaf(acc[i][j][r], f, -rf.y) - lo[i]) - (lab == (uint32_t)r ? 1.f : 0.f);
                                t[r] += __float_as_int(rf.w) >= 0 && (plain || ((live[j] >> r) & 1u)) ? q * z * gr[i] : 0.f;
                            }
                        }
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            t[r] += __shfl_xor(t[r], 1);
                            t[r] += __shfl_xor(t[r], 2);
                            t[r] += __shfl_xor(t[r], 4);
                            t[r] += __shfl_xor(t[r], 8);
                            const uint32_t c = cl + j * 16u + r;
                            if ((lane & 15u) == 0 && c < g.n) g.tpart[(size_t)(tm * S::WM + wm) * g.n + c] = t[r];
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
#pragma unroll
                for (int i = 0; i < S::MT; ++i) {
                    const float4 rf = rows[(wm * S::MT + i) * 16u + (lane & 15u)];
                    const float f = rf.x * wsc;
                    const int32_t label = __float_as_int(rf.w);
                    const uint32_t lab = (uint32_t)(label - (int32_t)g.col0) - cl;
                    float v[S::NT][4];
                    if (plain) {
#pragma unroll
                        for (int j = 0; j < S::NT; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) v[j][r] = exp2_fast(fmaf(acc[i][j][r], f, -rf.y));
                    } else {
#pragma unroll
                        for (int j = 0; j < S::NT; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) v[j][r] = (live[j] >> r) & 1u ? exp2_fast(fmaf(acc[i][j][r], f, -rf.y)) : 0.f;
                    }
                    if (__any(lab < S::NT * 16u)) {
                        const float one = lab < S::NT * 16u && row0 + i * 16u < g.m ? exp2_fast(g.lo[row0 + i * 16u]) : 1.f;
#pragma unroll
                        for (int j = 0; j < S::NT; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (lab == j * 16u + r) v[j][r] -= one;
                    }
                    if (__any(label < 0)) {  // padding: whatever its query holds
#pragma unroll
                        for (int j = 0; j < S::NT; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) v[j][r] = label < 0 ? 0.f : v[j][r];
                    }
                    if constexpr (KIND == K_F32) {  // f32 probabilities carry every factor
                        f32x4 x[S::NT];
#pragma unroll
                        for (int j = 0; j < S::NT; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) x[j][r] = scaled ? v[j][r] * rf.z * h[j][r] : v[j][r] * rf.z;  // (v is 0 where h is)
                        store_lines<SCRATCH / 128>(scratch, x, reinterpret_cast<float*>(g.prob), g.prob_ld, row0 - (lane & 15u) + i * 16u, g.m, c0, g.prob_ld, lane);
                        continue;
                    }
                    ushort4 hi[S::NT], lo[S::NT];
                    if (KIND == K_BF16 && g.prob_kind == K_BF16) {
#pragma unroll
                        for (int j = 0; j < S::NT; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float x = g.h ? v[j][r] * rf.z * h[j][r] : v[j][r] * rf.z;
                                const uint16_t b = to_half<true>(x);
                                (&hi[j].x)[r] = b, (&lo[j].x)[r] = to_half<true>(x - from_half<true>(b));
                            }
                    } else
#pragma unroll
                    for (int j = 0; j < S::NT; ++j) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[j][r] *= rf.z;
                        hi[j].x = to_half<false>(v[j][0]), hi[j].y = to_half<false>(v[j][1]), hi[j].z = to_half<false>(v[j][2]), hi[j].w = to_half<false>(v[j][3]);
                        if (g.prob_planes > 1) {
                            lo[j].x = to_half<false>((v[j][0] - from_half<false>(hi[j].x)) * 2048.f), lo[j].y = to_half<false>((v[j][1] - from_half<false>(hi[j].y)) * 2048.f);
                            lo[j].z = to_half<false>((v[j][2] - from_half<false>(hi[j].z)) * 2048.f), lo[j].w = to_half<false>((v[j][3] - from_half<false>(hi[j].w)) * 2048.f);
                        }
                    }
                    store_lines<SCRATCH / 128>(scratch, hi, g.prob, g.prob_ld, row0 - (lane & 15u) + i * 16u, g.m, c0, g.prob_ld, lane);
                    if (g.prob_planes > 1) store_lines<SCRATCH / 128>(scratch, lo, g.prob + g.prob_plane, g.prob_ld, row0 - (lane & 15u) + i * 16u, g.m, c0, g.prob_ld, lane);
                    __builtin_amdgcn_sched_barrier(0);  // one block of rows at a time: interleaved, they do not fit the registers
                }
            }
        } else if constexpr (EPI == EPI_PART) {
            float* to = g.out_part + (size_t)sp * g.m * g.n;
#pragma unroll
            for (int i = 0; i < S::MT; ++i) store_lines<SCRATCH / 128>(scratch, acc[i], to, g.n, row0 - (lane & 15u) + i * 16u, g.m, c0, g.n, lane);  // (n: a multiple of 4)
        } else {
            const float wf = g.wf ? *g.wf : 1.f;
            const bool full = g.out_scalar == SC_F32, fits = g.n % 8u == 0 && g.out_ld % 8u == 0 && ((uintptr_t)g.out & 15u) == 0;
            const bool lines = !full && fits, wide = full && fits && (!g.tcoef || (g.raw_ld % 4u == 0 && ((uintptr_t)g.raw & 15u) == 0));
            if (wide) {
                constexpr bool AHEAD = S::MT <= 4;  // a block of rows ahead, or each one's reading is waited for (the large tile has no registers left)
                f32x4 less[2][4];
                if (AHEAD && g.tcoef) load_lines((const float*)g.raw, g.raw_ld, row0 - (lane & 15u), g.m, c0, g.n, lane, less[0]);
#pragma unroll
                for (int i = 0; i < S::MT; ++i) {
                    const uint32_t row = row0 + i * 16u;
                    const bool has = row < g.m;
                    const float rf = has && g.rf ? g.rf[row] * wf : wf;
                    f32x4 x[S::NT];
#pragma unroll
                    for (int j = 0; j < S::NT; ++j) x[j] = acc[i][j] * rf;
                    if (g.tcoef) {
                        const int next = AHEAD ? i + 1 : i;
                        if (next < S::MT) load_lines((const float*)g.raw, g.raw_ld, row0 - (lane & 15u) + next * 16u, g.m, c0, g.n, lane, less[next & 1]);
                        store_lines<SCRATCH / 128>(scratch, x, (float*)g.out, g.out_ld, row - (lane & 15u), g.m, c0, g.n, lane, less[i & 1], has ? g.tcoef[row] : 0.f,
                                                   has ? g.tinv[row] : 0.f);
                    } else store_lines<SCRATCH / 128>(scratch, x, (float*)g.out, g.out_ld, row - (lane & 15u), g.m, c0, g.n, lane);
                }
                continue;
            }
#pragma unroll
            for (int i = 0; i < S::MT; ++i) {
                const uint32_t row = row0 + i * 16u;
                const bool has = row < g.m;
                const float rf = has && g.rf ? g.rf[row] * wf : wf;
                const float tc = has && g.tcoef ? g.tcoef[row] : 0.f, ti = has && g.tcoef ? g.tinv[row] : 0.f;
                ushort4 o[S::NT];
#pragma unroll
                for (int j = 0; j < S::NT; ++j) {
                    const uint32_t c = cl + j * 16u;
                    f32x4 v = acc[i][j] * rf;
                    if (tc != 0.f && c < g.n) v -= load4(g.raw, g.raw_scalar, (uint64_t)row * g.raw_ld + c, g.n - c) * ti * tc;  // (in this order: 1 / |row|^2 may not exist in f32)
                    if (lines) o[j] = to_half4(g.out_scalar, v);
                    else if (has && c < g.n) store4(g.out, g.out_scalar, (uint64_t)row * g.out_ld + c, v, g.n - c);
                }
                if (lines) store_lines<SCRATCH / 128>(scratch, o, (uint16_t*)g.out, g.out_ld, row0 - (lane & 15u) + i * 16u, g.m, c0, g.n, lane);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the loads beyond the last step: LDS is given back with nothing on its way into it)
}

}  // namespace learn
}  // namespace vs
