// learn.hip -- libvs_learn.so (include/vs_learn.h): the softmax loss of queries over all rows of a table or index and its gradients
// (products on the matrix pipe, learn_product.hpp), rows read by number and their gradient.
#include "../../include/vs_learn.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "learn_lookup.hpp"
#include "learn_product.hpp"

namespace vs {
namespace learn {

thread_local std::string g_err;
struct Fail {
    int code;
    std::string msg;
};
[[noreturn]] static void fail(int code, std::string msg) { throw Fail{code, std::move(msg)}; }
static void need(bool cond, const char* what) {
    if (!cond) fail(VS_ERR_INVALID_ARGUMENT, what);
}
static void hip_ok(hipError_t e, const char* what) {
    if (e != hipSuccess) fail(VS_ERR_DEVICE, std::string(what) + ": " + hipGetErrorString(e));
}
static void launched(const char* what) { hip_ok(hipGetLastError(), what); }

// ------------------------------------------------------------------------------------------------ preparation kernels
// Number formats.  Both sides bf16: the operands are used as they are (bf16 products are exact in f32).  Both sides f16, inner product: the
// same on the f16 pipe.  Everything else (f32 anywhere, mixed types, f16 under cosine) is split into f16 planes, x = hi + lo with hi = f16(x),
// lo = f16(x - hi): 22 bits of x.  Three of the four products of two such numbers are summed (lo lo is below 2^-22 of the result), which is
// f32's accuracy at three times the f16 product's cost -- the matrix pipe's f32 product costs sixteen.  (A few f32 queries of f32 rows are
// multiplied as f32 all the same, probabilities included: the time is the rows' reading then; kFullQueries.)  f16's narrow range is met by
// powers of two: a query row, the rows of a piece of the table (inner product), or the normalised vector (cosine) is scaled so that its
// largest element lies in [2^12, 2^13]; what is 2^-36 of the largest is lost.
// The gradients' products are f16 for every type: the probabilities are numbers this code rounds itself, and in bf16 their rounding would be
// as large as the result's (measured at 4,096 x 131,072 x 768: 0.0025 of the gradient against 0.0017 for one rounding of the exact one).  One
// f16 (2^-11) under a bf16 result, two under f16 and f32 ones (the second times 2^11: a probability below f16's normal range keeps its bits);
// bf16 rows and queries are exact in a scaled f16.  (For a few bf16 queries, two bf16 and the rows as they are: kFewQueries.)

struct QueryPrep {
    const void* q;
    int scalar;
    uint64_t ld;
    uint32_t n, d, dp;
    const void* labels;
    uint32_t label_bytes;
    uint32_t rows;                 // labels beyond are ignored
    const uint64_t* keys;          // labels of removed members too
    float scale;
    uint32_t cosine, raw;          // raw: the operands are the values themselves
    int kind, gkind;               // K_*: of the scores' operands, of the gradients'
    bool wide;                     // 16-byte aligned rows
    void* planes;                  // nullptr: read in place
    void* gplanes;                 // f32, bf16: the queries as an operand of dw, or nullptr
    uint32_t nplanes;
    uint64_t plane;
    uint32_t* tops;                // the pieces' largest elements, zeroed for rows_top_kernel
    uint32_t pieces;
    int32_t* label;
    float4* row;  // the products' factors: (zf, lse2, pf 2^-lo, label)
    // backward (g != nullptr)
    const float* g;
    const float* lse;
    float *df, *inv, *lo;
    int32_t *ge, *xe;
};

constexpr int32_t kNoExponent = -1000000;

__device__ __forceinline__ int32_t exponent_of(float x) {  // x < 2^e (0, infinities and NaN: 0)
    if (!(x > 0.f) || x == __builtin_inff()) return 0;
    int e;
    (void)frexpf(x, &e);
    return e;
}

// eight consecutive values of a row into its planes (to: element `at` of the first)
__device__ __forceinline__ void put_planes(void* planes, uint64_t at, uint64_t plane, uint32_t nplanes, int kind, const float (&x)[8]) {
    if (kind == K_F32) {
        store8(planes, SC_F32, at, 8, true, x);
        return;
    }
    const bool bf = kind == K_BF16;
    uint16_t* to = reinterpret_cast<uint16_t*>(planes) + at;
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (bf) {
            hi[r] = (uint32_t)to_half<true>(x[2 * r]) | (uint32_t)to_half<true>(x[2 * r + 1]) << 16;
            lo[r] = 0;
        } else {
            const uint16_t a = to_half<false>(x[2 * r]), b = to_half<false>(x[2 * r + 1]);
            hi[r] = (uint32_t)a | (uint32_t)b << 16;
            lo[r] = (uint32_t)to_half<false>(x[2 * r] - from_half<false>(a)) | (uint32_t)to_half<false>(x[2 * r + 1] - from_half<false>(b)) << 16;
        }
    }
    *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (nplanes > 1) *reinterpret_cast<uint4*>(to + plane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}
// sum of squares and largest |element| of a row, by `lanes` lanes (a power of two, up to a wave)
__device__ __forceinline__ void row_extent(const void* p, int scalar, uint64_t at, uint32_t d, bool wide, uint32_t lane, uint32_t lanes, float& ss, float& top) {
    ss = 0.f, top = 0.f;
    for (uint32_t k = lane * 8u; k < d; k += lanes * 8u) {
        float x[8];
        load8(p, scalar, at + k, d - k, wide, x);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            ss = fmaf(x[r], x[r], ss);
            top = fmaxf(top, fabsf(x[r]));
        }
    }
    for (uint32_t o = lanes >> 1; o; o >>= 1) {
        ss += __shfl_xor(ss, (int)o);
        top = fmaxf(top, __shfl_xor(top, (int)o));
    }
}

// one wave per query: its norm, largest element, factors, and its planes
__global__ __launch_bounds__(256) void query_prep_kernel(QueryPrep a) {
    if (blockIdx.x == 0)
        for (uint32_t x = threadIdx.x; x < a.pieces; x += 256) a.tops[x] = 0;
    const uint32_t lane = threadIdx.x & 63u, i = blockIdx.x * 4u + (threadIdx.x >> 6);
    if (i >= a.n) return;
    float ss = 0.f, top = 0.f;
    if (a.cosine || !a.raw || (a.g && a.gkind == K_F16)) row_extent(a.q, a.scalar, (uint64_t)i * a.ld, a.d, a.wide, lane, 64, ss, top);
    const float inv = !a.cosine ? 1.f : ss > 0.f ? 1.f / sqrtf(ss) : 0.f;
    const int32_t e = a.raw || a.cosine ? 0 : exponent_of(top);
    const bool unit = a.cosine && a.kind == K_F32;  // (the planes hold the direction)
    int64_t y = a.label_bytes == 8 ? reinterpret_cast<const int64_t*>(a.labels)[i] : reinterpret_cast<const int32_t*>(a.labels)[i];
    if (y < 0 || y >= (int64_t)a.rows || (a.keys && a.keys[y] == ~0ull)) y = -1;
    const float g = a.g && y >= 0 ? a.g[i] : 0.f;
    if (a.gplanes) {  // as grad_queries_kernel; f32: with the factors themselves, bf16: the probabilities carry them
        const bool on = y >= 0 && g != 0.f, full = a.gkind == K_F32;
        const float f = g * a.scale;
        for (uint32_t k = lane * 8u; k < a.dp; k += 512) {
            float x[8];
            load8(a.q, a.scalar, (uint64_t)i * a.ld + k, on && k < a.d ? a.d - k : 0u, a.wide, x);
#pragma unroll
            for (int r = 0; r < 8; ++r) x[r] = !on ? 0.f : full ? x[r] * inv * f : x[r];
            put_planes(a.gplanes, (uint64_t)i * a.dp + k, 0, 1, a.gkind, x);
        }
    }
    if (a.planes) {
        for (uint32_t k = lane * 8u; k < a.dp; k += 512) {
            float x[8];
            load8(a.q, a.scalar, (uint64_t)i * a.ld + k, k < a.d ? a.d - k : 0u, a.wide, x);
            if (!a.raw || unit) {
#pragma unroll
                for (int r = 0; r < 8; ++r) x[r] = a.cosine ? x[r] * (inv * (unit ? 1.f : 8192.f)) : ldexpf(x[r], 13 - e);
            }
            put_planes(a.planes, (uint64_t)i * a.dp + k, a.plane, a.nplanes, a.kind, x);
        }
    }
    if (lane) return;
    a.label[i] = (int32_t)y;
    const float s2 = a.scale * kLog2e;
    float4 row = make_float4(unit ? s2 : a.raw ? s2 * inv : a.cosine ? s2 * 0x1p-26f : ldexpf(s2, e - 13), 0.f, 0.f, __int_as_float((int32_t)y));
    if (a.g) {
        // lse in base-2 units, in two parts: row.y and what its rounding lost, which goes into the factor
        const float lse = a.lse[i];
        row.y = lse * kLog2e;
        const float lo = fabsf(row.y) < __builtin_inff() ? fmaf(lse, kLog2e, -row.y) + lse * kLog2eLo : 0.f;
        a.lo[i] = lo;
        a.inv[i] = inv;
        // f16 probabilities: (p - [label]) * m * 2^15 with g = m * 2^x, 1/2 <= |m| < 1: below 2^15, off by at most 2^-11 of themselves or 2^-39
        // f32: the probability itself times the row's inverse length; the query's factors go to dq and, in front of dw, to the query.  bf16, whose
        // queries and rows are used as they are: times all of them.
        int x = 0;
        const float m = frexpf(g, &x);
        row.z = (a.gkind == K_F32 ? 1.f : a.gkind == K_BF16 ? g * a.scale * inv : m * 32768.f) * exp2f(-lo);
        a.df[i] = y < 0 ? 0.f : a.gkind == K_F32 ? g * a.scale * inv : a.gkind == K_BF16 ? 1.f : ldexpf(a.scale * (a.cosine ? inv * 0x1p-13f : 1.f), x - 15);
        a.ge[i] = x;
        a.xe[i] = y < 0 || !(g != 0.f) ? kNoExponent : x + exponent_of(a.cosine ? top * inv : top);
    }
    a.row[i] = row;
}

// The queries as an operand of dw = P^T q, in f16: rows of padding are zero whatever they held, every other row carries the power of two of its
// loss gradient, relative to the largest; *wf undoes it.
struct GradQueries {
    const void* q;
    int scalar;
    uint64_t ld;
    uint32_t n, d, dp, cosine, nplanes;
    bool wide;
    const int32_t *label, *ge, *xe;
    const float* inv;
    float scale;
    void* planes;
    uint64_t plane;
    int32_t* top;  // [1]
    float* wf;     // [1]
};
// (the largest exponent: every workgroup looks for itself where the queries are few, which saves a launch)
constexpr uint32_t kOwnExponent = 8192;
__device__ __forceinline__ int32_t grad_exponent(const GradQueries& a) {
    __shared__ int32_t red[16];
    int32_t top = kNoExponent;
    for (uint32_t i = threadIdx.x; i < a.n; i += blockDim.x) top = max(top, a.xe[i]);
    for (int o = 32; o; o >>= 1) top = max(top, __shfl_xor(top, o));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    top = red[0];
    for (uint32_t x = 1; x < blockDim.x / 64; ++x) top = max(top, red[x]);
    return top == kNoExponent ? 0 : top;
}
__global__ __launch_bounds__(1024) void grad_exponent_kernel(GradQueries a) {
    const int32_t top = grad_exponent(a);
    if (threadIdx.x == 0) a.top[0] = top;
}
__global__ __launch_bounds__(256) void grad_queries_kernel(GradQueries a) {
    const int32_t top = a.n <= kOwnExponent ? grad_exponent(a) : a.top[0];
    if (blockIdx.x == 0 && threadIdx.x == 0) a.wf[0] = ldexpf(a.scale, top - 28);
    const uint32_t lane = threadIdx.x & 63u, i = blockIdx.x * 4u + (threadIdx.x >> 6);
    if (i >= a.n) return;
    const bool on = a.label[i] >= 0 && a.xe[i] != kNoExponent;  // (padding, and queries whose loss nobody asks about)
    const int32_t up = a.ge[i] - top + 13;
    const float inv = a.cosine ? a.inv[i] : 1.f;
    for (uint32_t k = lane * 8u; k < a.dp; k += 512) {
        float x[8];
        load8(a.q, a.scalar, (uint64_t)i * a.ld + k, on && k < a.d ? a.d - k : 0u, a.wide, x);
#pragma unroll
        for (int r = 0; r < 8; ++r) x[r] = ldexpf(x[r] * inv, up);
        put_planes(a.planes, (uint64_t)i * a.dp + k, a.plane, a.nplanes, K_F16, x);
    }
}

struct RowPrep {
    const void* w;        // the piece's first row
    int scalar;
    uint64_t ld;
    uint32_t rows, d, dp;
    const uint64_t* keys;  // of the piece
    uint32_t cosine, raw, nplanes;
    int kind;
    bool wide;
    void* planes;
    uint64_t plane;
    uint32_t* top;   // bits of the largest |element| of the piece (inner product planes)
    float* wsc;      // 2^(e - 13)
    float* inv;      // 1 / |row|
};
template <int SC>
__global__ __launch_bounds__(256) void rows_top_kernel(RowPrep a) {
    const uint32_t lane = threadIdx.x & 63u;
    float top = 0.f;
    const auto take = [&](uint64_t at, uint32_t left, bool wide) {
        float x[8];
        load8(a.w, SC, at, left, wide, x);
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (fabsf(x[r]) < __builtin_inff()) top = fmaxf(top, fabsf(x[r]));
    };
    if (a.ld == a.d && !a.keys) {  // one stretch of memory
        const uint64_t all = (uint64_t)a.rows * a.d;
        const bool wide = ((uintptr_t)a.w & 15u) == 0;
        for (uint64_t k = ((uint64_t)blockIdx.x * 256u + threadIdx.x) * 8u; k < all; k += (uint64_t)gridDim.x * 2048u) take(k, all - k < 8 ? (uint32_t)(all - k) : 8u, wide);
    } else {
        for (uint32_t j = blockIdx.x * 4u + (threadIdx.x >> 6); j < a.rows; j += gridDim.x * 4u) {
            if (a.keys && a.keys[j] == ~0ull) continue;
            for (uint32_t k = lane * 8u; k < a.d; k += 512) take((uint64_t)j * a.ld + k, a.d - k, a.wide);
        }
    }
    __shared__ float red[4];
    top = wave_max(top);
    if (lane == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    if (threadIdx.x == 0 && top > 0.f) atomicMax(a.top, __float_as_uint(top));  // (a maximum: the same bits whatever the order)
}
// `lanes` lanes per row of the piece (8 .. 64: as many as a short row has pieces of 8 elements)
template <int SC>
__global__ __launch_bounds__(256) void rows_planes_kernel(RowPrep a, uint32_t lanes) {
    const uint32_t lane = threadIdx.x & (lanes - 1u), j = blockIdx.x * (256u / lanes) + threadIdx.x / lanes;
    const int32_t e = a.raw || a.cosine ? 0 : exponent_of(__uint_as_float(*a.top));
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.wsc) *a.wsc = a.raw || a.cosine ? 1.f : ldexpf(1.f, e - 13);
    if (j >= a.rows) return;
    const bool live = !(a.keys && a.keys[j] == ~0ull);
    float inv = 1.f;
    if (a.cosine && !a.raw) {
        float ss, top;
        row_extent(a.w, SC, (uint64_t)j * a.ld, a.d, a.wide, lane, lanes, ss, top);
        inv = live && ss > 0.f ? 1.f / sqrtf(ss) : 0.f;
        if (lane == 0 && a.inv) a.inv[j] = inv;
    }
    for (uint32_t k = lane * 8u; k < a.dp; k += lanes * 8u) {
        float x[8];
        load8(a.w, SC, (uint64_t)j * a.ld + k, live && k < a.d ? a.d - k : 0u, a.wide, x);
        if (!a.raw) {
#pragma unroll
            for (int r = 0; r < 8; ++r) x[r] = a.cosine ? x[r] * (inv * 8192.f) : ldexpf(x[r], 13 - e);
        }
        put_planes(a.planes, (uint64_t)j * a.dp + k, a.plane, a.nplanes, a.kind, x);
    }
}
// 1 / |row| of a table whose rows are used as they are
__global__ __launch_bounds__(256) void rows_inverse_norm_kernel(const void* w, int scalar, uint64_t ld, uint32_t rows, uint32_t d, bool wide, float* inv) {
    const uint32_t lane = threadIdx.x & 63u, j = blockIdx.x * 4u + (threadIdx.x >> 6);
    if (j >= rows) return;
    float ss, top;
    row_extent(w, scalar, (uint64_t)j * ld, d, wide, lane, 64, ss, top);
    if (lane == 0) inv[j] = ss > 0.f ? 1.f / sqrtf(ss) : 0.f;
}
// ------------------------------------------------------------------------------------------------ joins
// natural logarithm of 2^x y, rounded once
__device__ __forceinline__ float log_sum(float2 a) { return (float)(((double)a.x + log2((double)a.y)) * 0.69314718055994530942); }
__global__ __launch_bounds__(256) void loss_join_kernel(const float2* part, uint32_t part_ld, uint32_t n, const int32_t* label, const float2* zlab,
                                                        float* loss, float* lse) {
    __shared__ float2 red[4];
    const uint32_t i = blockIdx.x, lane = threadIdx.x & 63u;
    float2 a = make_float2(-__builtin_inff(), 0.f);
    for (uint32_t t = threadIdx.x; t < part_ld; t += 256) a = join_sums(a, part[(size_t)i * part_ld + t]);
    for (int o = 1; o < 64; o <<= 1) a = join_sums(a, make_float2(__shfl_xor(a.x, o), __shfl_xor(a.y, o)));
    if (lane == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x) return;
    for (int x = 1; x < 4; ++x) a = join_sums(a, red[x]);
    if (label[i] < 0) {
        lse[i] = log_sum(a);
        loss[i] = 0.f;
        return;
    }
    // a: all columns but the label's
    // (what the label's score lost when it was rounded is half a step of lse: dropped, it is the largest error of p - 1 near p = 1)
    const float2 zy = zlab[i];
    const float apart = a.x - zy.x - zy.y;
    lse[i] = log_sum(join_sums(a, make_float2(zy.x, exp2f(zy.y))));
    loss[i] = apart < 64.f ? log1pf(a.y * exp2f(apart)) : (apart + log2f(a.y)) * kLn2;
}

// dq of one query: slices of k in order, pieces in order; after the last piece its factor, the way through the normalisation, the cast
struct QueryJoin {
    const float* part;   // [splits][n][dn]
    uint32_t splits, n, d, dn;
    const float* wsc;
    float* acc;          // [n][dn]
    uint32_t first, last, cosine;
    const float *df, *inv;
    const void* q;
    int scalar;
    uint64_t ld;
    void* out;
    uint64_t out_ld;
};
__global__ __launch_bounds__(256) void query_join_kernel(QueryJoin a) {
    __shared__ float red[4];
    const uint32_t i = blockIdx.x;
    const float wsc = a.wsc ? *a.wsc : 1.f, df = a.last ? a.df[i] : 1.f, inv = a.last && a.cosine ? a.inv[i] : 0.f;
    float dot = 0.f;
    for (uint32_t k = threadIdx.x; k < a.d; k += 256) {
        float s = 0.f;
        for (uint32_t x0 = 0; x0 < a.splits; x0 += 16) {  // (sixteen loads on their way at a time)
            float v[16];
#pragma unroll
            for (uint32_t x = 0; x < 16; ++x) v[x] = x0 + x < a.splits ? a.part[((size_t)(x0 + x) * a.n + i) * a.dn + k] : 0.f;
#pragma unroll
            for (uint32_t x = 0; x < 16; ++x) s += v[x];
        }
        s *= wsc;
        if (!a.first) s += a.acc[(size_t)i * a.dn + k];
        if (a.last && !a.cosine) {
            store_scalar(a.out, a.scalar, (uint64_t)i * a.out_ld + k, df == 0.f ? 0.f : s * df);
            continue;
        }
        if (a.last) {
            s *= df;
            dot = fmaf(s, load_scalar(a.q, a.scalar, (uint64_t)i * a.ld + k) * inv, dot);
        }
        a.acc[(size_t)i * a.dn + k] = s;
    }
    if (!a.last || !a.cosine) return;
    dot = wave_sum(dot);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = dot;
    __syncthreads();
    dot = (red[0] + red[1]) + (red[2] + red[3]);
    for (uint32_t k = threadIdx.x; k < a.d; k += 256)  // (each thread reads what it wrote itself)
        store_scalar(a.out, a.scalar, (uint64_t)i * a.out_ld + k,
                     df == 0.f ? 0.f : a.acc[(size_t)i * a.dn + k] - load_scalar(a.q, a.scalar, (uint64_t)i * a.ld + k) * inv * dot);
}
// cosine: what dw_j has along w_j / |w_j|: sum over queries of g c z, / |w_j|
__global__ __launch_bounds__(256) void row_along_kernel(const float* tpart, uint32_t parts, uint32_t n, const float* inv, float* coef) {
    const uint32_t j = blockIdx.x * 256u + threadIdx.x;
    if (j >= n) return;
    float s = 0.f;
    for (uint32_t x = 0; x < parts; ++x) s += tpart[(size_t)x * n + j];
    coef[j] = s * kLn2 * inv[j];
}

// ------------------------------------------------------------------------------------------------ host side
template <class S, int FORM, int EPI, int KIND>
static void run_product(const ProductArgs& g, hipStream_t st) {
    static std::atomic<uint64_t> allowed{0};  // a bit per device
    int device = 0;
    hip_ok(hipGetDevice(&device), "device");
    if (device >= 64 || !(allowed.load(std::memory_order_relaxed) >> device & 1u)) {
        hip_ok(hipFuncSetAttribute(reinterpret_cast<const void*>(&product_kernel<S, FORM, EPI, KIND>), hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS),
               "shared memory of the product");
        if (device < 64) allowed.fetch_or(1ull << device, std::memory_order_relaxed);
    }
    const uint64_t tiles = (uint64_t)g.tiles_m * g.tiles_n * g.splits;
    if (tiles >= (1ull << 31)) fail(VS_ERR_UNSUPPORTED, "too many tiles");
    constexpr uint32_t resident = 256u * (160u * 1024u / S::LDS);
    hipLaunchKernelGGL((product_kernel<S, FORM, EPI, KIND>), dim3((uint32_t)std::min<uint64_t>((tiles + 7) / 8 * 8, resident)), dim3(S::NW * 64), S::LDS, st, g);
    launched("product");
}
enum : int { LARGE = 0, MEDIUM = 1, SMALL = 2, SLIM = 3 };
constexpr uint32_t kTileM[4] = {Large::TM, Medium::TM, Small::TM, Slim::TM}, kTileN[4] = {Large::TN, Medium::TN, Small::TN, Slim::TN};
constexpr uint32_t kWaveRows[4] = {Large::WM, Medium::WM, Small::WM, Slim::WM};
template <int FORM, int EPI, int KIND>
static void product_of(const ProductArgs& g, int shape, hipStream_t st) {
    switch (shape) {
        case LARGE: return run_product<Large, FORM, EPI, KIND>(g, st);
        case MEDIUM: return run_product<Medium, FORM, EPI, KIND>(g, st);
        default: return run_product<Small, FORM, EPI, KIND>(g, st);
    }
}
template <int FORM, int EPI>
static void product(ProductArgs g, int shape, int kind, hipStream_t st) {
    g.tiles_m = (g.m + kTileM[shape] - 1) / kTileM[shape];
    g.tiles_n = (g.n + kTileN[shape] - 1) / kTileN[shape];
    if (kind == K_F32) {
        if constexpr (FORM != DW) {
            if (shape == SLIM) return run_product<Slim, FORM, EPI, K_F32>(g, st);
        }
        return run_product<Small, FORM, EPI, K_F32>(g, st);
    }
    if (kind == K_BF16) return product_of<FORM, EPI, K_BF16>(g, shape, st);
    product_of<FORM, EPI, K_F16>(g, shape, st);
}
// The tile for m x n outputs: the one whose rounds over the chip take least.  A round of large tiles (256 workgroups) is 1, of medium ones
// 0.62, of small ones (512) 0.44 -- measured over 64 .. 4,096 x 131,072 outputs, 768 and 1,536 deep: 256 x 32,768 in 26.6 / 19.5 / 23.7 us,
// 300 x 131,072 in 89 / 79 / 91, 777 x 131,072 in 167 / 177 / 229, 64 x 131,072 in 52 / 36 / 32.  `whole`: k is sliced until the chip is
// full, so only the outputs beyond m and n are waste.
static int choose_shape(uint64_t m, uint64_t n, bool whole) {
    const double round[3] = {1.0, 0.62, 0.44};
    const uint64_t resident[3] = {256, 256, 512};
    int best = SMALL;
    double least = 1e300;
    for (int x = 0; x < 3; ++x) {
        const uint64_t tiles = ((m + kTileM[x] - 1) / kTileM[x]) * ((n + kTileN[x] - 1) / kTileN[x]);
        const double cost = round[x] * (whole ? (double)tiles / resident[x] : (double)((tiles + resident[x] - 1) / resident[x]));
        if (cost < least) best = x, least = cost;
    }
    return best;
}

struct Rows {  // vs_rows resolved
    const char* data = nullptr;
    int scalar = 0;
    size_t rows = 0, dim = 0, ld = 0;  // ld in elements
    const uint64_t* keys = nullptr;    // only where members were removed
    const float* inv = nullptr;
    int metric = -1, device = -1;
};
static size_t size_of(int scalar) { return scalar == VS_SCALAR_F32 ? 4 : 2; }
static void need_scalar(int scalar, const char* what) {
    if (scalar != VS_SCALAR_F32 && scalar != VS_SCALAR_F16 && scalar != VS_SCALAR_BF16) fail(VS_ERR_UNSUPPORTED, std::string(what) + ": f32, f16 or bf16");
}
static Rows resolve(const vs_rows* r) {
    need(r, "null rows");
    Rows o;
    if (r->index) {
        vs_hnsw_row_view v;
        const int rc = vs_hnsw_rows(r->index, &v);
        if (rc != VS_OK) fail(rc, vs_hnsw_last_error());
        need_scalar(v.quantization, "rows of an index");
        o.data = (const char*)v.d_rows;
        o.scalar = v.quantization;
        o.rows = v.slots;
        o.dim = v.dimensions;
        o.ld = v.stride_bytes / size_of(v.quantization);
        o.keys = v.removed ? v.d_keys : nullptr;
        o.inv = v.d_inverse_norms;
        o.metric = v.metric;
        o.device = v.device;
    } else {
        need_scalar(r->scalar, "rows");
        need(r->rows == 0 || r->d_data, "null rows");
        need(r->stride >= r->dim, "rows: stride below the dimension");
        o.data = (const char*)r->d_data;
        o.scalar = r->scalar;
        o.rows = r->rows;
        o.dim = r->dim;
        o.ld = r->stride;
    }
    need(o.dim > 0, "dimension must be > 0");
    if (o.rows >= (1ull << 31) || o.dim > (1u << 16) || o.ld > (1u << 20)) fail(VS_ERR_UNSUPPORTED, "rows: below 2^31 of them, up to 65,536 elements, strides up to 2^20");
    return o;
}
// The index's device is current for the duration of a call.
struct OnDevice {
    int before = -1;
    explicit OnDevice(int device) {
        if (device < 0) return;
        hip_ok(hipGetDevice(&before), "device");
        if (before == device) before = -1;
        else hip_ok(hipSetDevice(device), "device");
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

struct Layout {  // offsets into the caller's scratch
    size_t at = 0;
    size_t take(size_t bytes) {
        const size_t r = at;
        at += (bytes + 255) & ~(size_t)255;
        return r;
    }
};

// What a loss call does, from sizes, types, alignment and what is asked of it.
struct Plan {
    Rows w;
    uint32_t n = 0, v = 0, d = 0, dp = 0;
    bool cosine = false, raw = false, q_in_place = false, w_in_place = false;
    bool inv_own = false, inv_scores = false;  // the rows' inverse lengths are computed here; by the scores' product
    bool grad_q = false, grad_w = false;
    int kind = K_F16, gkind = K_F16;                    // operands of the scores; of the gradients' products
    uint32_t es = 2, ges = 2, bk = 64, gbk = 64;        // bytes per element and elements per step of both
    bool regrow = false;                                // the rows of dq are laid out apart from those of the scores
    uint32_t nq = 1, nw = 1, np = 1, nqg = 1, nwg = 1;  // planes of the queries, the rows, the probabilities, the queries of dw, the rows of dq
    uint32_t piece = 0, pieces = 0;
    int shape_s = LARGE, shape_q = LARGE, shape_w = LARGE;  // of the scores, dq, dw
    uint32_t splits = 1, qsteps = 1, tiles_v = 0, trows = 0;
    size_t o_label, o_row, o_qplanes, o_top, o_wsc, o_inv, o_wplanes, o_gwplanes, o_part, o_zlab;
    size_t o_df, o_qinv, o_lo, o_ge, o_xe, o_exp, o_gplanes, o_prob, o_tpart, o_coef, o_qpart, o_qacc;
    size_t bytes = 0;
};

// Re-laid rows and probabilities of one piece.  A step of 4,096 x 131,072 x 768 took 3.66 / 3.45 / 3.43 / 3.40 ms with 256 / 640 / 1,400 / 2,400 MiB:
// larger pieces leave fewer CUs without a tile, and what the last-level cache (256 MiB) no longer holds costs about as much.
constexpr size_t kPieceBytes = 640ull << 20;
constexpr size_t kSplitBytes = 128ull << 20;    // f32 slices of dq
// Up to this many f32 queries of f32 rows are multiplied as f32: the rows are then read once where the split re-lays them first, about four times
// the traffic, and the f32 MFMA's sixteenth of the f16 rate does not show before more queries than that.  60,000 x 768, as f32 / split, loss and
// gradients: 40 queries 67 + 217 / 159 + 304 us, 72: 125 + 350 / 165 + 301, 128: 120 + 352 / 164 + 306; by cosine 64: 72 + 253 / 132 +
// 342, 72 (with the lengths in a pass of their own): 144 + 392 / 137 + 309.  (One limit for the loss and its gradient: a probability near 1 is
// only as good as the two agree on its score.)
constexpr uint32_t kFullQueries = 64;
// Up to this many bf16 queries of bf16 rows the probabilities are kept as two bf16, times all factors, instead of one f16: the gradients' products
// then use rows and queries as they are -- twice the products, but the rows need not be laid out in f16 first.  Gradients of 64 x
// 60,000 x 768 161 -> 125 us, 128: 184 / 136, 256: 219 / 185, 256 x 100,000 x 1536 595 / 573, by cosine 782 / 792.
constexpr uint32_t kFewQueries = 256;

// Rows per piece, at most `most`.  A workgroup per CU owns 256 x 256 outputs, so 257 tiles take as long as 512: of the sizes allowed, the one
// whose products leave the fewest CUs idle (in steps of 64 k; a tile's epilogue counts 6, a piece's launches 10).
static size_t piece_rows(uint64_t n, uint64_t v, uint64_t d, size_t most, bool grad_w) {
    if (most >= v) return (v + 255) / 256 * 256;
    const uint64_t tm = (n + 255) / 256, td = (d + 255) / 256, all = (v + 255) / 256;
    const auto cost = [&](uint64_t c) {
        return (tm * c + 255) / 256 * ((d + 63) / 64 + 6) + (grad_w ? (c * td + 255) / 256 * ((n + 63) / 64 + 6) : 0) + 10;
    };
    const uint64_t top = std::max<uint64_t>(1, most / 256);
    uint64_t best = top, best_cost = ~0ull;
    for (uint64_t c = std::max<uint64_t>(1, top / 3); c <= top; ++c) {
        const uint64_t whole = all / c, rest = all % c, total = whole * cost(c) + (rest ? cost(rest) : 0);
        if (total <= best_cost) best = c, best_cost = total;
    }
    return best * 256;
}

static Plan plan(const vs_rows* rows, const vs_softmax* q, bool grad_q, bool grad_w) {
    Plan p;
    p.w = resolve(rows);
    need(q, "null queries");
    need_scalar(q->scalar, "queries");
    need(q->n == 0 || (q->d_queries && q->d_labels), "null queries or labels");
    need(q->label_bytes == 4 || q->label_bytes == 8, "labels: 4 or 8 bytes");
    need(q->stride >= p.w.dim, "queries: stride below the dimension");
    need(q->metric == VS_METRIC_IP || q->metric == VS_METRIC_COS, "a loss needs the inner product or the cosine");
    need(p.w.metric < 0 || p.w.metric == q->metric, "the loss's metric is not the index's");
    need(std::isfinite(q->scale), "scale must be finite");
    if (q->n > (1u << 20) || q->stride > (1u << 20)) fail(VS_ERR_UNSUPPORTED, "queries: up to 2^20 of them, strides up to 2^20");
    const uint32_t n = p.n = (uint32_t)q->n, v = p.v = (uint32_t)p.w.rows, d = p.d = (uint32_t)p.w.dim;
    p.dp = (d + 63u) & ~63u;
    p.cosine = q->metric == VS_METRIC_COS;
    const int tq = q->scalar, tw = p.w.scalar;
    const bool bf = tq == VS_SCALAR_BF16 && tw == VS_SCALAR_BF16, full = tq == VS_SCALAR_F32 && tw == VS_SCALAR_F32 && n <= kFullQueries;
    p.kind = full ? K_F32 : bf ? K_BF16 : K_F16;
    p.gkind = full ? K_F32 : bf && n <= kFewQueries ? K_BF16 : K_F16;
    p.es = full ? 4 : 2, p.bk = 128 / p.es;
    p.ges = p.es, p.gbk = p.bk;
    p.raw = full || bf || (tq == VS_SCALAR_F16 && tw == VS_SCALAR_F16 && !p.cosine);
    const uint32_t line = 16 / p.es;
    p.q_in_place = p.raw && !(full && p.cosine) && d % line == 0 && q->stride % line == 0 && (uintptr_t)q->d_queries % 16 == 0;
    p.w_in_place = p.raw && !p.w.keys && d % line == 0 && p.w.ld % line == 0 && (uintptr_t)p.w.data % 16 == 0;
    p.inv_own = p.cosine && !(p.raw && p.w.inv);
    p.inv_scores = full && p.inv_own;
    p.nq = !p.raw && (p.cosine || tq == VS_SCALAR_F32) ? 2 : 1;
    p.nw = !p.raw && (p.cosine || tw == VS_SCALAR_F32) ? 2 : 1;
    p.grad_q = grad_q;
    p.grad_w = grad_w;
    const bool grad = grad_q || grad_w;
    p.np = p.gkind == K_BF16 || (!full && ((grad_q && tq != VS_SCALAR_BF16) || (grad_w && tw != VS_SCALAR_BF16))) ? 2 : 1;
    p.nqg = !full && tw != VS_SCALAR_BF16 && (p.cosine || tq == VS_SCALAR_F32) ? 2 : 1;
    p.regrow = bf && grad_q && p.gkind == K_F16;
    p.nwg = p.regrow ? 1 : p.nw;
    // pieces of the table: one, unless rows are re-laid or probabilities are kept for the two products that read them
    const size_t per_row = (p.w_in_place ? 0 : (size_t)p.nw * p.dp * p.es) + (p.regrow ? (size_t)p.dp * 2 : 0) + (grad ? (size_t)p.np * n * p.ges : 0);
    size_t piece = v;
    if (per_row) piece = std::min<size_t>(v, std::max<size_t>(2048, kPieceBytes / per_row));
    piece = std::min<size_t>(piece, 1u << 20);
    if (piece) {
        piece = piece_rows(n, v, d, piece, grad_w);
        p.pieces = (uint32_t)((v + piece - 1) / piece);
    }
    p.piece = (uint32_t)piece;
    const int few = n <= 32 ? SLIM : SMALL;  // (one query against 300,000 x 768: 300 us by small tiles, 210 by slim ones; 20 against 10,000 x 128 the same)
    p.shape_s = full ? few : choose_shape(n, piece, false);
    p.shape_w = full ? SMALL : choose_shape(piece, d, false);
    p.shape_q = full ? few : choose_shape(n, d, true);
    const size_t qtiles = (size_t)((n + kTileM[p.shape_q] - 1) / kTileM[p.shape_q]) * ((d + kTileN[p.shape_q] - 1) / kTileN[p.shape_q]);
    const size_t dn = (d + 3u) & ~3u;
    const uint32_t ksteps = (uint32_t)std::max<size_t>(1, (piece + p.gbk - 1) / p.gbk);
    if (grad_q && n) {
        size_t s = std::max<size_t>(1, (p.shape_q == SLIM ? 768 : p.shape_q == SMALL ? 512 : 256) / qtiles);
        s = std::min<size_t>(s, std::max<size_t>(1, kSplitBytes / (n * dn * 4)));
        s = std::min<size_t>(s, std::max<uint32_t>(1, ksteps / 4));
        p.qsteps = (uint32_t)((ksteps + s - 1) / s);
        p.splits = (ksteps + p.qsteps - 1) / p.qsteps;
    }
    const uint32_t stn = kTileN[p.shape_s], stm = kTileM[p.shape_s];
    p.tiles_v = p.pieces ? (p.pieces - 1) * (p.piece / stn) + (uint32_t)((v - (size_t)(p.pieces - 1) * p.piece + stn - 1) / stn) : 0;
    p.trows = (n + stm - 1) / stm * kWaveRows[p.shape_s];
    Layout l;
    p.o_label = l.take((size_t)n * 4);
    p.o_row = l.take((size_t)n * 16);
    p.o_qplanes = l.take(p.q_in_place ? 0 : (size_t)p.nq * n * p.dp * p.es);
    p.o_top = l.take((size_t)p.pieces * 4);
    p.o_wsc = l.take((size_t)p.pieces * 4);
    p.o_inv = l.take(p.inv_own ? (size_t)v * 4 : 0);
    p.o_wplanes = l.take(p.w_in_place ? 0 : (size_t)p.nw * piece * p.dp * p.es);
    p.o_gwplanes = l.take(p.regrow ? piece * p.dp * 2 : 0);
    if (!grad) {
        p.o_part = l.take((size_t)n * p.tiles_v * 8);
        p.o_zlab = l.take((size_t)n * 8);
    } else {
        p.o_df = l.take((size_t)n * 4);
        p.o_qinv = l.take((size_t)n * 4);
        p.o_lo = l.take((size_t)n * 4);
        p.o_ge = l.take((size_t)n * 4);
        p.o_xe = l.take((size_t)n * 4);
        p.o_exp = l.take(8);
        p.o_gplanes = l.take(grad_w ? (size_t)p.nqg * n * p.dp * p.ges : 0);
        p.o_prob = l.take((size_t)p.np * n * (((size_t)piece + 7) & ~(size_t)7) * p.ges);
        p.o_tpart = l.take(grad_w && p.cosine ? (size_t)p.trows * piece * 4 : 0);
        p.o_coef = l.take(grad_w && p.cosine ? (size_t)piece * 4 : 0);
        p.o_qpart = l.take(grad_q ? (size_t)p.splits * n * dn * 4 : 0);
        p.o_qacc = l.take(grad_q && (p.pieces > 1 || p.cosine) ? (size_t)n * dn * 4 : 0);
    }
    p.bytes = l.at;
    return p;
}

// Which planes are multiplied: (lo hi, hi lo, hi hi) of what there is -- the largest products last, so that the small ones are added to small
// sums --, or hi hi alone.
static void plane_pairs(ProductArgs& g, uint32_t na, uint32_t nb, bool all) {
    g.segs = 0;
    g.seg_a = g.seg_b = 0;
    if (all && na > 1) g.seg_a |= 1u << (4 * g.segs++);
    if (all && nb > 1) g.seg_b |= 1u << (4 * g.segs++);
    ++g.segs;
}

struct Call {  // what the two calls share
    const Plan& p;
    const vs_softmax& q;
    char* work;
    hipStream_t st;
    template <class T>
    T* at(size_t o) const { return reinterpret_cast<T*>(work + o); }

    void queries(const float* lse, const float* g) const {
        QueryPrep a = {};
        a.q = q.d_queries;
        a.scalar = q.scalar;
        a.ld = q.stride;
        a.n = p.n, a.d = p.d, a.dp = p.dp;
        a.labels = q.d_labels;
        a.label_bytes = (uint32_t)q.label_bytes;
        a.rows = p.v;
        a.keys = p.w.keys;
        a.scale = q.scale;
        a.cosine = p.cosine, a.raw = p.raw, a.kind = p.kind, a.gkind = p.gkind;
        a.wide = wide_rows(a.q, a.scalar, a.ld);
        a.planes = p.q_in_place ? nullptr : at<char>(p.o_qplanes);
        a.nplanes = p.nq;
        a.plane = (uint64_t)p.n * p.dp;
        a.tops = at<uint32_t>(p.o_top);
        a.pieces = p.pieces;
        a.label = at<int32_t>(p.o_label);
        a.row = at<float4>(p.o_row);
        if (g) {
            a.g = g;
            a.lse = lse;
            a.df = at<float>(p.o_df), a.inv = at<float>(p.o_qinv), a.lo = at<float>(p.o_lo);
            a.ge = at<int32_t>(p.o_ge), a.xe = at<int32_t>(p.o_xe);
            a.gplanes = p.grad_w && p.gkind != K_F16 ? at<char>(p.o_gplanes) : nullptr;
        }
        hipLaunchKernelGGL(query_prep_kernel, dim3((p.n + 3) / 4), dim3(256), 0, st, a);
        launched("queries");
    }
    void tables() const {  // once per call, before the pieces
        if (p.raw && p.inv_own && !p.inv_scores) {
            hipLaunchKernelGGL(rows_inverse_norm_kernel, dim3((p.v + 3) / 4), dim3(256), 0, st, p.w.data, p.w.scalar, (uint64_t)p.w.ld, p.v, p.d,
                               wide_rows(p.w.data, p.w.scalar, p.w.ld), at<float>(p.o_inv));
            launched("norms");
        }
    }
    const float* h() const { return !p.cosine || !p.raw ? nullptr : p.w.inv ? p.w.inv : at<float>(p.o_inv); }       // score factor of a column
    const float* inv() const { return p.raw && p.w.inv ? p.w.inv : at<float>(p.o_inv); }
    template <int SC>
    void launch_rows(const RowPrep& a) const {
        if (!a.raw && !p.cosine) {
            const uint64_t blocks = ((uint64_t)a.rows * a.d + 8191) / 8192;  // (four loads per thread; few workgroups: each ends in an atomic on one word)
            hipLaunchKernelGGL((rows_top_kernel<SC>), dim3((uint32_t)std::min<uint64_t>(1024, blocks)), dim3(256), 0, st, a);
            launched("rows");
        }
        uint32_t lanes = 8;
        while (lanes < 64 && lanes * 16 <= a.dp) lanes *= 2;
        const uint32_t per = 256 / lanes;
        hipLaunchKernelGGL((rows_planes_kernel<SC>), dim3((a.rows + per - 1) / per), dim3(256), 0, st, a, lanes);
        launched("rows");
    }
    // a piece's rows re-laid: as they are (raw: bf16 or f16), or as f16 planes
    Operand relay(uint32_t x, uint32_t first, uint32_t count, size_t o_planes, uint32_t nplanes, bool raw) const {
        RowPrep a = {};
        a.w = p.w.data + (size_t)first * p.w.ld * size_of(p.w.scalar);
        a.scalar = p.w.scalar;
        a.ld = p.w.ld;
        a.rows = count, a.d = p.d, a.dp = p.dp;
        a.keys = p.w.keys ? p.w.keys + first : nullptr;
        a.cosine = p.cosine, a.raw = raw, a.kind = raw ? p.kind : K_F16, a.nplanes = nplanes;
        a.wide = wide_rows(a.w, a.scalar, a.ld);
        a.planes = at<char>(o_planes);
        a.plane = (uint64_t)p.piece * p.dp;
        a.top = at<uint32_t>(p.o_top) + x;
        a.wsc = at<float>(p.o_wsc) + x;
        a.inv = p.cosine && !p.raw ? at<float>(p.o_inv) + first : nullptr;
        switch (p.w.scalar) {
            case VS_SCALAR_F32: launch_rows<SC_F32>(a); break;
            case VS_SCALAR_F16: launch_rows<SC_F16>(a); break;
            default: launch_rows<SC_BF16>(a); break;
        }
        const uint64_t es = raw ? p.es : 2;
        return Operand{(const char*)a.planes, a.plane * es, (uint64_t)p.dp * es, count, p.dp};
    }
    // the piece's rows as an operand of the scores; of dq
    Operand rows(uint32_t x, uint32_t first, uint32_t count) const {
        if (p.w_in_place) return Operand{p.w.data + (size_t)first * p.w.ld * size_of(p.w.scalar), 0, p.w.ld * p.es, count, p.d};
        return relay(x, first, count, p.o_wplanes, p.nw, p.raw);
    }
    Operand grad_rows(const Operand& scores, uint32_t x, uint32_t first, uint32_t count) const {
        return p.regrow ? relay(x, first, count, p.o_gwplanes, 1, false) : scores;
    }
    // scores of all queries against a piece: operands and factors
    ProductArgs scores(const Operand& w, uint32_t x, uint32_t first, uint32_t count) const {
        ProductArgs g = {};
        g.a = p.q_in_place ? Operand{(const char*)q.d_queries, 0, q.stride * p.es, p.n, p.d}
                           : Operand{at<char>(p.o_qplanes), (uint64_t)p.n * p.dp * p.es, (uint64_t)p.dp * p.es, p.n, p.dp};
        g.b = w;
        g.m = p.n, g.n = count;
        g.k = std::min(g.a.cols, g.b.cols);  // (a re-laid operand's padding is zero)
        g.splits = 1;
        g.ksteps = (g.k + p.bk - 1) / p.bk;
        plane_pairs(g, p.nq, p.nw, true);
        g.row = at<float4>(p.o_row);
        g.norms = p.inv_scores ? at<float>(p.o_inv) + first : nullptr;
        g.h = h() && !p.inv_scores ? h() + first : nullptr;
        g.wsc = p.raw || p.cosine ? nullptr : at<float>(p.o_wsc) + x;
        g.keys = p.w.keys ? p.w.keys + first : nullptr;
        g.col0 = first;
        return g;
    }
};

static void need_work(const Plan& p, const void* work, size_t bytes) {
    need(bytes >= p.bytes && (p.bytes == 0 || work), "d_work is smaller than the call needs");
    need((uintptr_t)work % 256 == 0, "d_work must be 256-byte aligned");
}

static void loss(const vs_rows* rows, const vs_softmax* q, float* d_loss, float* d_lse, void* work, size_t work_bytes, hipStream_t st) {
    const Plan p = plan(rows, q, false, false);
    if (!p.n) return;
    need(d_loss && d_lse, "null outputs");
    need_work(p, work, work_bytes);
    OnDevice dev(p.w.device);
    const Call c{p, *q, (char*)work, st};
    c.queries(nullptr, nullptr);
    if (p.v) c.tables();
    uint32_t tile = 0;
    for (uint32_t x = 0; x < p.pieces; ++x) {
        const uint32_t first = x * p.piece, count = std::min(p.piece, p.v - first);
        const Operand w = c.rows(x, first, count);
        ProductArgs g = c.scores(w, x, first, count);
        g.part = c.at<float2>(p.o_part);
        g.part_ld = p.tiles_v;
        g.part0 = tile;
        g.zlab = c.at<float2>(p.o_zlab);
        product<SCORES, EPI_LOSS>(g, p.shape_s, p.kind, st);
        tile += (count + kTileN[p.shape_s] - 1) / kTileN[p.shape_s];
    }
    hipLaunchKernelGGL(loss_join_kernel, dim3(p.n), dim3(256), 0, st, c.at<float2>(p.o_part), p.tiles_v, p.n, c.at<int32_t>(p.o_label),
                       c.at<float2>(p.o_zlab), d_loss, d_lse);
    launched("join");
}

static void loss_grad(const vs_rows* rows, const vs_softmax* q, const float* d_lse, const float* d_g, void* d_gq, size_t gq_ld, void* d_gw, size_t gw_ld,
                      void* work, size_t work_bytes, hipStream_t st) {
    const Plan p = plan(rows, q, d_gq != nullptr, d_gw != nullptr);
    if (!d_gq && !d_gw) return;
    need(!d_gq || gq_ld >= p.d, "gradient of the queries: stride below the dimension");
    need(!d_gw || gw_ld >= p.d, "gradient of the rows: stride below the dimension");
    need(p.n == 0 || (d_lse && d_g), "null lse or gradient of the loss");
    need_work(p, work, work_bytes);
    OnDevice dev(p.w.device);
    if (!p.n || !p.v) {  // nothing to learn from: the gradients there are are zero
        if (d_gq && p.n) launch_zero_rows(d_gq, q->scalar, gq_ld, p.n, p.d, st);
        if (d_gw && p.v) launch_zero_rows(d_gw, p.w.scalar, gw_ld, p.v, p.d, st);
        launched("zero");
        return;
    }
    const Call c{p, *q, (char*)work, st};
    c.queries(d_lse, d_g);
    c.tables();
    const uint64_t gplane = (uint64_t)p.n * p.dp;
    const Operand gq = {c.at<char>(p.o_gplanes), gplane * p.ges, (uint64_t)p.dp * p.ges, p.n, p.dp};
    if (d_gw && p.gkind == K_F16) {
        GradQueries a = {};
        a.q = q->d_queries;
        a.scalar = q->scalar;
        a.ld = q->stride;
        a.n = p.n, a.d = p.d, a.dp = p.dp, a.cosine = p.cosine, a.nplanes = p.nqg;
        a.wide = wide_rows(a.q, a.scalar, a.ld);
        a.label = c.at<int32_t>(p.o_label), a.ge = c.at<int32_t>(p.o_ge), a.xe = c.at<int32_t>(p.o_xe);
        a.inv = c.at<float>(p.o_qinv);
        a.scale = q->scale;
        a.planes = c.at<char>(p.o_gplanes);
        a.plane = gplane;
        a.top = c.at<int32_t>(p.o_exp);
        a.wf = c.at<float>(p.o_exp) + 1;
        if (p.n > kOwnExponent) hipLaunchKernelGGL(grad_exponent_kernel, dim3(1), dim3(1024), 0, st, a);
        hipLaunchKernelGGL(grad_queries_kernel, dim3((p.n + 3) / 4), dim3(256), 0, st, a);
        launched("queries");
    }
    const uint32_t dn = (p.d + 3u) & ~3u;
    for (uint32_t x = 0; x < p.pieces; ++x) {
        const uint32_t first = x * p.piece, count = std::min(p.piece, p.v - first);
        const Operand w = c.rows(x, first, count);
        ProductArgs g = c.scores(w, x, first, count);
        g.lo = c.at<float>(p.o_lo);
        g.prob = c.at<uint16_t>(p.o_prob);
        g.prob_ld = (count + 7u) & ~7u;
        g.prob_plane = (uint64_t)p.n * g.prob_ld;
        g.prob_planes = p.np;
        g.prob_kind = p.gkind;
        g.tpart = d_gw && p.cosine ? c.at<float>(p.o_tpart) : nullptr;
        g.graw = d_g;
        if (g.tpart) product<SCORES, EPI_PROB_ALONG>(g, p.shape_s, p.kind, st);
        else product<SCORES, EPI_PROB>(g, p.shape_s, p.kind, st);
        const Operand prob{(const char*)g.prob, g.prob_plane * p.ges, (uint64_t)g.prob_ld * p.ges, p.n, g.prob_ld};
        if (d_gq) {
            ProductArgs b = {};
            b.a = prob;
            b.b = c.grad_rows(w, x, first, count);
            b.m = p.n, b.n = dn, b.k = count;
            b.splits = p.splits;
            b.ksteps = p.qsteps;
            const bool both = q->scalar != VS_SCALAR_BF16 || p.gkind == K_BF16;
            plane_pairs(b, p.np, p.nwg, both);
            b.lo_first = both && p.np > 1;
            b.out_part = c.at<float>(p.o_qpart);
            product<DQ, EPI_PART>(b, p.shape_q, p.gkind, st);
            QueryJoin j = {};
            j.part = b.out_part;
            j.splits = p.splits, j.n = p.n, j.d = p.d, j.dn = dn;
            j.wsc = (p.raw && !p.regrow) || p.cosine ? nullptr : c.at<float>(p.o_wsc) + x;
            j.acc = c.at<float>(p.o_qacc);
            j.first = x == 0, j.last = x + 1 == p.pieces, j.cosine = p.cosine;
            j.df = c.at<float>(p.o_df), j.inv = c.at<float>(p.o_qinv);
            j.q = q->d_queries, j.scalar = q->scalar, j.ld = q->stride;
            j.out = d_gq, j.out_ld = gq_ld;
            hipLaunchKernelGGL(query_join_kernel, dim3(p.n), dim3(256), 0, st, j);
            launched("join");
        }
        if (d_gw) {
            if (p.cosine) {
                hipLaunchKernelGGL(row_along_kernel, dim3((count + 255) / 256), dim3(256), 0, st, g.tpart, p.trows, count, c.inv() + first,
                                   c.at<float>(p.o_coef));
                launched("rows");
            }
            ProductArgs b = {};
            b.a = prob;
            b.b = gq;
            b.m = count, b.n = p.d, b.k = p.n;
            b.splits = 1;
            b.ksteps = (p.n + p.gbk - 1) / p.gbk;
            const bool both = p.w.scalar != VS_SCALAR_BF16 || p.gkind == K_BF16;
            plane_pairs(b, p.np, p.nqg, both);
            b.lo_first = both && p.np > 1;
            b.out = (char*)d_gw + (size_t)first * gw_ld * size_of(p.w.scalar);
            b.out_scalar = p.w.scalar;
            b.out_ld = gw_ld;
            b.wf = p.gkind != K_F16 ? nullptr : c.at<float>(p.o_exp) + 1;
            b.rf = p.cosine && p.gkind == K_F16 ? c.inv() + first : nullptr;
            b.tcoef = p.cosine ? c.at<float>(p.o_coef) : nullptr;
            b.tinv = p.cosine ? c.inv() + first : nullptr;
            b.raw = p.w.data + (size_t)first * p.w.ld * size_of(p.w.scalar);
            b.raw_scalar = p.w.scalar;
            b.raw_ld = p.w.ld;
            product<DW, EPI_ROWS>(b, p.shape_w, p.gkind, st);
        }
    }
}

template <class F>
static int guarded(F&& f) {
    try {
        f();
        return VS_OK;
    } catch (const Fail& x) {
        g_err = x.msg;
        return x.code;
    } catch (const std::exception& x) {
        g_err = x.what();
        return VS_ERR_DEVICE;
    } catch (...) {
        g_err = "unknown error";
        return VS_ERR_DEVICE;
    }
}

}  // namespace learn
}  // namespace vs

using namespace vs::learn;

extern "C" {

const char* vs_learn_last_error(void) { return g_err.c_str(); }

int vs_lookup_device(const vs_rows* rows, const void* d_ids, size_t id_bytes, size_t n, float scale, void* d_out, int out_scalar, size_t out_stride, void* stream) {
    return guarded([&] {
        const Rows r = resolve(rows);
        need_scalar(out_scalar, "output");
        need(id_bytes == 4 || id_bytes == 8, "ids: 4 or 8 bytes");
        need(out_stride >= r.dim, "output: stride below the dimension");
        if (!n) return;
        need(d_ids && d_out, "null ids or output");
        if (n >= (1ull << 31)) fail(VS_ERR_UNSUPPORTED, "below 2^31 ids");
        OnDevice dev(r.device);
        launch_lookup(r.data, r.scalar, r.ld, (uint32_t)r.rows, (uint32_t)r.dim, r.keys, d_ids, (uint32_t)id_bytes, (uint32_t)n, scale, d_out, out_scalar, out_stride,
                      (hipStream_t)stream);
        launched("lookup");
    });
}

size_t vs_lookup_grad_work(size_t n, size_t rows, size_t dim) { return lookup_grad_layout(n, rows, dim).bytes; }

int vs_lookup_grad_device(const void* d_grad, int grad_scalar, size_t grad_stride, const void* d_ids, size_t id_bytes, size_t n, size_t rows, size_t dim, float scale,
                          int accumulate, void* d_out, int out_scalar, size_t out_stride, void* d_work, size_t work_bytes, void* stream) {
    return guarded([&] {
        need_scalar(grad_scalar, "gradient");
        need_scalar(out_scalar, "output");
        need(id_bytes == 4 || id_bytes == 8, "ids: 4 or 8 bytes");
        need(dim > 0 && grad_stride >= dim && out_stride >= dim, "a stride is below the dimension");
        if (!rows) return;
        need(d_out, "null output");
        need(n == 0 || (d_grad && d_ids), "null gradient or ids");
        if (n >= (1ull << 30) || rows >= (1ull << 31) - 1 || dim > (1u << 16)) fail(VS_ERR_UNSUPPORTED, "below 2^30 ids, 2^31 rows, up to 65,536 elements");
        const LookupGradLayout l = lookup_grad_layout(n, rows, dim);
        need(work_bytes >= l.bytes && (l.bytes == 0 || d_work), "d_work is smaller than the call needs");
        need((uintptr_t)d_work % 256 == 0, "d_work must be 256-byte aligned");
        launch_lookup_grad(d_grad, grad_scalar, grad_stride, d_ids, (uint32_t)id_bytes, (uint32_t)n, (uint32_t)rows, (uint32_t)dim, scale, accumulate != 0, d_out, out_scalar,
                           out_stride, l, (char*)d_work, (hipStream_t)stream);
        launched("lookup gradient");
    });
}

size_t vs_softmax_loss_work(const vs_rows* rows, const vs_softmax* q) {
    size_t bytes = 0;
    return guarded([&] { bytes = plan(rows, q, false, false).bytes; }) == VS_OK ? bytes : 0;
}
int vs_softmax_loss_device(const vs_rows* rows, const vs_softmax* q, float* d_loss, float* d_lse, void* d_work, size_t work_bytes, void* stream) {
    return guarded([&] { loss(rows, q, d_loss, d_lse, d_work, work_bytes, (hipStream_t)stream); });
}
size_t vs_softmax_loss_grad_work(const vs_rows* rows, const vs_softmax* q, int queries, int table) {
    size_t bytes = 0;
    return guarded([&] { bytes = plan(rows, q, queries != 0, table != 0).bytes; }) == VS_OK ? bytes : 0;
}
int vs_softmax_loss_grad_device(const vs_rows* rows, const vs_softmax* q, const float* d_lse, const float* d_grad_loss, void* d_grad_queries,
                                size_t grad_queries_stride, void* d_grad_rows, size_t grad_rows_stride, void* d_work, size_t work_bytes, void* stream) {
    return guarded([&] {
        loss_grad(rows, q, d_lse, d_grad_loss, d_grad_queries, grad_queries_stride, d_grad_rows, grad_rows_stride, d_work, work_bytes, (hipStream_t)stream);
    });
}

}  // extern "C"
