// learn_lookup.hpp -- rows read by number, and the gradient that goes back to them.
//
// Forward: out[t] = scale * row[id[t]].  Bound by the memory: one 16-byte piece of a row per thread and load.
//
// Backward: sums over the t that read a row, in the order of t, without float atomics (two calls give the same bits).  The (id, t) pairs are
// sorted by id -- stable, so t ascends within an id --, the sorted list is cut into runs of kRun entries, a workgroup sums each run: an id
// whose entries all lie in one run is written at once, the others leave a partial row at the run's head (the id began earlier) or tail
// (it goes on), and a second kernel adds those up from the run where the id begins.  An id read n times costs n / kRun serial steps, not n.
#pragma once
#include <hip/hip_runtime.h>

#include "learn_device.hpp"

namespace vs {
namespace learn {

__device__ __forceinline__ int64_t load_id(const void* ids, uint32_t bytes, uint64_t t) {
    return bytes == 8 ? reinterpret_cast<const int64_t*>(ids)[t] : (int64_t) reinterpret_cast<const int32_t*>(ids)[t];
}

// eight consecutive elements as floats / from floats; `left` of them exist
__device__ __forceinline__ void load8(const void* p, int scalar, uint64_t i, uint32_t left, bool wide, float (&v)[8]) {
    if (wide && left >= 8) {
        if (scalar == SC_F32) {
            const f32x4 a = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p) + i)[0], b = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p) + i)[1];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = a[r], v[4 + r] = b[r];
        } else {
            const uint4 a = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (scalar == SC_F16) v[2 * r] = from_half<false>((uint16_t)w[r]), v[2 * r + 1] = from_half<false>((uint16_t)(w[r] >> 16));
                else v[2 * r] = from_half<true>((uint16_t)w[r]), v[2 * r + 1] = from_half<true>((uint16_t)(w[r] >> 16));
            }
        }
        return;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] = (uint32_t)r < left ? load_scalar(p, scalar, i + r) : 0.f;
}
__device__ __forceinline__ void store8(void* p, int scalar, uint64_t i, uint32_t left, bool wide, const float (&v)[8]) {
    if (wide && left >= 8) {
        if (scalar == SC_F32) {
            f32x4* to = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p) + i);
            to[0] = f32x4{v[0], v[1], v[2], v[3]};
            to[1] = f32x4{v[4], v[5], v[6], v[7]};
        } else {
            uint32_t w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (scalar == SC_F16) w[r] = (uint32_t)to_half<false>(v[2 * r]) | (uint32_t)to_half<false>(v[2 * r + 1]) << 16;
                else w[r] = (uint32_t)to_half<true>(v[2 * r]) | (uint32_t)to_half<true>(v[2 * r + 1]) << 16;
            }
            *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r)
        if ((uint32_t)r < left) store_scalar(p, scalar, i + r, v[r]);
}
inline bool wide_rows(const void* p, int scalar, uint64_t ld) {
    const uint64_t e = scalar == SC_F32 ? 4 : 2;
    return (uintptr_t)p % 16 == 0 && ld * e % 16 == 0;
}

struct LookupArgs {
    const void* rows;
    int scalar;
    uint64_t ld;
    uint32_t count, dim, chunks;  // chunks: 8-element pieces of a row
    const uint64_t* keys;
    const void* ids;
    uint32_t id_bytes, n;
    float scale;
    void* out;
    int out_scalar;
    uint64_t out_ld;
    bool wide_in, wide_out;
};
__global__ __launch_bounds__(256) void lookup_kernel(LookupArgs a) {
    const uint64_t total = (uint64_t)a.n * a.chunks;
    for (uint64_t x = (uint64_t)blockIdx.x * 256u + threadIdx.x; x < total; x += (uint64_t)gridDim.x * 256u) {
        const uint32_t t = (uint32_t)(x / a.chunks), k = (uint32_t)(x - (uint64_t)t * a.chunks) * 8u;
        const int64_t id = load_id(a.ids, a.id_bytes, t);
        float v[8];
        if (id >= 0 && id < (int64_t)a.count && !(a.keys && a.keys[id] == kFreeKey)) {
            load8(a.rows, a.scalar, (uint64_t)id * a.ld + k, a.dim - k, a.wide_in, v);
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] *= a.scale;
        } else {
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] = 0.f;
        }
        store8(a.out, a.out_scalar, (uint64_t)t * a.out_ld + k, a.dim - k, a.wide_out, v);
    }
}
inline void launch_lookup(const void* rows, int scalar, uint64_t ld, uint32_t count, uint32_t dim, const uint64_t* keys, const void* ids, uint32_t id_bytes, uint32_t n,
                          float scale, void* out, int out_scalar, uint64_t out_ld, hipStream_t st) {
    LookupArgs a = {rows, scalar, ld, count, dim, (dim + 7) / 8, keys, ids, id_bytes, n, scale, out, out_scalar, out_ld, wide_rows(rows, scalar, ld), wide_rows(out, out_scalar, out_ld)};
    const uint64_t blocks = ((uint64_t)n * a.chunks + 255) / 256;
    hipLaunchKernelGGL(lookup_kernel, dim3((uint32_t)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, st, a);
}

__global__ __launch_bounds__(256) void zero_rows_kernel(void* out, int scalar, uint64_t ld, uint32_t n, uint32_t dim, uint32_t chunks, bool wide) {
    const uint64_t total = (uint64_t)n * chunks;
    const float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (uint64_t x = (uint64_t)blockIdx.x * 256u + threadIdx.x; x < total; x += (uint64_t)gridDim.x * 256u) {
        const uint32_t t = (uint32_t)(x / chunks), k = (uint32_t)(x - (uint64_t)t * chunks) * 8u;
        store8(out, scalar, (uint64_t)t * ld + k, dim - k, wide, v);
    }
}
inline void launch_zero_rows(void* out, int scalar, uint64_t ld, uint32_t n, uint32_t dim, hipStream_t st) {
    const uint32_t chunks = (dim + 7) / 8;
    const uint64_t blocks = ((uint64_t)n * chunks + 255) / 256;
    hipLaunchKernelGGL(zero_rows_kernel, dim3((uint32_t)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, st, out, scalar, ld, n, dim, chunks, wide_rows(out, scalar, ld));
}

// ------------------------------------------------------------------------------------------------ stable sort of (id, t) by id
// Least significant digit first, kDigit bits a pass.  A wave owns kWaveItems consecutive entries: it counts its digits (first kernel), the
// counts of all waves are summed up digit by digit (second kernel, one workgroup), and it moves its entries to their places in order (third
// kernel: entries of one digit keep their order because the lanes of a wave rank themselves by lane number and the waves by position).
constexpr uint32_t kDigit = 9, kBins = 1u << kDigit, kWaveItems = 1024, kRun = 32;

struct SortArgs {
    const void* ids;
    uint32_t id_bytes, n, rows;    // ids beyond the rows sort last as `rows`
    uint32_t first, shift;         // first pass: keys come from ids
    const uint32_t *key_in, *pos_in;
    uint32_t *key_out, *pos_out;
    uint32_t* counts;              // [kBins][waves]
    uint32_t waves;
};
__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, uint32_t t) {
    if (!a.first) return a.key_in[t];
    const int64_t id = load_id(a.ids, a.id_bytes, t);
    return id >= 0 && id < (int64_t)a.rows ? (uint32_t)id : a.rows;
}
__global__ __launch_bounds__(64) void sort_count_kernel(SortArgs a) {
    __shared__ uint32_t bins[kBins];
    const uint32_t lane = threadIdx.x, t0 = blockIdx.x * kWaveItems, t1 = min(a.n, t0 + kWaveItems);
    for (uint32_t b = lane; b < kBins; b += 64) bins[b] = 0;
    __syncthreads();
    for (uint32_t t = t0 + lane; t < t1; t += 64) atomicAdd(&bins[(sort_key(a, t) >> a.shift) & (kBins - 1)], 1u);
    __syncthreads();
    for (uint32_t b = lane; b < kBins; b += 64) a.counts[(size_t)b * a.waves + blockIdx.x] = bins[b];
}
// exclusive sums of kBins * waves counts, in place
__global__ __launch_bounds__(1024) void sort_sums_kernel(uint32_t* counts, uint32_t n) {
    __shared__ uint32_t part[1024];
    const uint32_t each = (n + 1023) / 1024, t0 = min(n, threadIdx.x * each), t1 = min(n, t0 + each);
    uint32_t s = 0;
    for (uint32_t t = t0; t < t1; ++t) s += counts[t];
    part[threadIdx.x] = s;
    __syncthreads();
    for (uint32_t o = 1; o < 1024; o <<= 1) {
        const uint32_t add = threadIdx.x >= o ? part[threadIdx.x - o] : 0;
        __syncthreads();
        part[threadIdx.x] += add;
        __syncthreads();
    }
    uint32_t at = threadIdx.x ? part[threadIdx.x - 1] : 0;
    for (uint32_t t = t0; t < t1; ++t) {
        const uint32_t c = counts[t];
        counts[t] = at;
        at += c;
    }
}
__global__ __launch_bounds__(64) void sort_move_kernel(SortArgs a) {
    __shared__ uint32_t at[kBins];
    const uint32_t lane = threadIdx.x, t0 = blockIdx.x * kWaveItems, t1 = min(a.n, t0 + kWaveItems);
    for (uint32_t b = lane; b < kBins; b += 64) at[b] = a.counts[(size_t)b * a.waves + blockIdx.x];
    __syncthreads();
    for (uint32_t t = t0; t < t1; t += 64) {
        const bool on = t + lane < t1;
        const uint32_t key = on ? sort_key(a, t + lane) : 0u, digit = (key >> a.shift) & (kBins - 1);
        uint64_t same = __ballot(on);
#pragma unroll
        for (uint32_t b = 0; b < kDigit; ++b) {
            const uint64_t m = __ballot((digit >> b) & 1u);
            same &= (digit >> b) & 1u ? m : ~m;
        }
        const uint32_t rank = mbcnt(same);
        const uint32_t to = on ? at[digit] + rank : 0u;
        __syncthreads();
        if (on && rank == 0) at[digit] += (uint32_t)__popcll(same);
        __syncthreads();
        if (on) {
            a.key_out[to] = key;
            a.pos_out[to] = a.first ? t + lane : a.pos_in[t + lane];
        }
    }
}

// ------------------------------------------------------------------------------------------------ sums of the runs
struct RunArgs {
    const uint32_t *key, *pos;
    uint32_t n, rows, dim, chunks, runs;
    const void* grad;
    int grad_scalar;
    uint64_t grad_ld;
    float scale;
    uint32_t accumulate;
    void* out;
    int out_scalar;
    uint64_t out_ld;
    float* part;  // [runs][2][chunks * 8]: sums of the id that began earlier; of the id that goes on
    bool wide_in, wide_out;
};
__device__ __forceinline__ void finish_row(const RunArgs& a, uint32_t row, uint32_t k, float (&v)[8]) {
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] *= a.scale;
    if (a.accumulate) {
        float o[8];
        load8(a.out, a.out_scalar, (uint64_t)row * a.out_ld + k, a.dim - k, a.wide_out, o);
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] += o[r];
    }
    store8(a.out, a.out_scalar, (uint64_t)row * a.out_ld + k, a.dim - k, a.wide_out, v);
}
// one workgroup per run; a thread owns 8 columns and goes through the run's entries
__global__ __launch_bounds__(256) void run_sums_kernel(RunArgs a) {
    __shared__ uint32_t key[kRun], pos[kRun];
    __shared__ uint32_t before, after;  // ids on both sides of the run
    const uint32_t t0 = blockIdx.x * kRun, m = min(kRun, a.n - t0);
    if (threadIdx.x < m) key[threadIdx.x] = a.key[t0 + threadIdx.x], pos[threadIdx.x] = a.pos[t0 + threadIdx.x];
    if (threadIdx.x == 64) before = t0 ? a.key[t0 - 1] : ~0u;
    if (threadIdx.x == 65) after = t0 + m < a.n ? a.key[t0 + m] : ~0u;
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < a.chunks; c += 256) {
        const uint32_t k = c * 8u;
        float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        uint32_t from = 0;
        for (uint32_t t = 0; t < m; ++t) {
            const uint32_t id = key[t];
            if (id >= a.rows) break;  // ids out of range sort last
            float v[8];
            load8(a.grad, a.grad_scalar, (uint64_t)pos[t] * a.grad_ld + k, a.dim - k, a.wide_in, v);
#pragma unroll
            for (int r = 0; r < 8; ++r) s[r] += v[r];
            const uint32_t next = t + 1 < m ? key[t + 1] : after;
            if (t + 1 < m && next == id) continue;
            const bool began = from == 0 && before == id, goes_on = t + 1 == m && next == id;
            if (began || goes_on) {
                float* to = a.part + ((size_t)blockIdx.x * 2u + (began ? 0u : 1u)) * (a.chunks * 8u) + k;
                reinterpret_cast<f32x4*>(to)[0] = f32x4{s[0], s[1], s[2], s[3]};
                reinterpret_cast<f32x4*>(to)[1] = f32x4{s[4], s[5], s[6], s[7]};
            } else {
                finish_row(a, id, k, s);
            }
            from = t + 1;
#pragma unroll
            for (int r = 0; r < 8; ++r) s[r] = 0.f;
        }
    }
}
// the run whose last id began in it and goes on: tail + heads of the following runs
__global__ __launch_bounds__(256) void run_join_kernel(RunArgs a) {
    const uint32_t t1 = (blockIdx.x + 1) * kRun;
    if (t1 >= a.n) return;
    const uint32_t id = a.key[t1 - 1], t0 = blockIdx.x * kRun;
    if (id >= a.rows || a.key[t1] != id) return;
    if (a.key[t0] == id && t0 && a.key[t0 - 1] == id) return;  // it began earlier: that run's workgroup adds up
    for (uint32_t c = threadIdx.x; c < a.chunks; c += 256) {
        const uint32_t k = c * 8u, w = a.chunks * 8u;
        const float* p = a.part + ((size_t)blockIdx.x * 2u + 1u) * w + k;
        float s[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) s[r] = p[r];
        for (uint32_t x = blockIdx.x + 1; x * kRun < a.n && a.key[x * kRun] == id; ++x) {
            const float* h = a.part + (size_t)x * 2u * w + k;
#pragma unroll
            for (int r = 0; r < 8; ++r) s[r] += h[r];
        }
        finish_row(a, id, k, s);
    }
}

struct LookupGradLayout {
    size_t key[2], pos[2], counts, part, bytes;
    uint32_t waves, runs, passes;
};
inline LookupGradLayout lookup_grad_layout(size_t n, size_t rows, size_t dim) {
    LookupGradLayout l = {};
    size_t at = 0;
    const auto take = [&](size_t b) {
        const size_t r = at;
        at += (b + 255) & ~(size_t)255;
        return r;
    };
    l.waves = (uint32_t)((n + kWaveItems - 1) / kWaveItems);
    l.runs = (uint32_t)((n + kRun - 1) / kRun);
    uint32_t bits = 1;
    while (bits < 31 && (rows >> bits)) ++bits;  // keys 0 .. rows
    l.passes = (bits + kDigit - 1) / kDigit;
    for (int x = 0; x < 2; ++x) l.key[x] = take(n * 4), l.pos[x] = take(n * 4);
    l.counts = take((size_t)l.waves * kBins * 4);
    l.part = take((size_t)l.runs * 2 * ((dim + 7) / 8 * 8) * 4);
    l.bytes = at;
    return l;
}
inline void launch_lookup_grad(const void* grad, int grad_scalar, uint64_t grad_ld, const void* ids, uint32_t id_bytes, uint32_t n, uint32_t rows, uint32_t dim, float scale,
                               bool accumulate, void* out, int out_scalar, uint64_t out_ld, const LookupGradLayout& l, char* work, hipStream_t st) {
    if (!accumulate) launch_zero_rows(out, out_scalar, out_ld, rows, dim, st);
    if (!n) return;
    SortArgs s = {};
    s.ids = ids;
    s.id_bytes = id_bytes;
    s.n = n;
    s.rows = rows;
    s.counts = (uint32_t*)(work + l.counts);
    s.waves = l.waves;
    uint32_t to = 0;
    for (uint32_t pass = 0; pass < l.passes; ++pass, to ^= 1u) {
        s.first = pass == 0;
        s.shift = pass * kDigit;
        s.key_in = (const uint32_t*)(work + l.key[to ^ 1u]), s.pos_in = (const uint32_t*)(work + l.pos[to ^ 1u]);
        s.key_out = (uint32_t*)(work + l.key[to]), s.pos_out = (uint32_t*)(work + l.pos[to]);
        hipLaunchKernelGGL(sort_count_kernel, dim3(l.waves), dim3(64), 0, st, s);
        hipLaunchKernelGGL(sort_sums_kernel, dim3(1), dim3(1024), 0, st, s.counts, l.waves * kBins);
        hipLaunchKernelGGL(sort_move_kernel, dim3(l.waves), dim3(64), 0, st, s);
    }
    to ^= 1u;
    RunArgs r = {};
    r.key = (const uint32_t*)(work + l.key[to]), r.pos = (const uint32_t*)(work + l.pos[to]);
    r.n = n, r.rows = rows, r.dim = dim, r.chunks = (dim + 7) / 8, r.runs = l.runs;
    r.grad = grad, r.grad_scalar = grad_scalar, r.grad_ld = grad_ld;
    r.scale = scale;
    r.accumulate = accumulate;
    r.out = out, r.out_scalar = out_scalar, r.out_ld = out_ld;
    r.part = (float*)(work + l.part);
    r.wide_in = wide_rows(grad, grad_scalar, grad_ld), r.wide_out = wide_rows(out, out_scalar, out_ld);
    hipLaunchKernelGGL(run_sums_kernel, dim3(l.runs), dim3(256), 0, st, r);
    hipLaunchKernelGGL(run_join_kernel, dim3(l.runs), dim3(256), 0, st, r);
}

}  // namespace learn
}  // namespace vs
