// learn_lookup.hpp -- rows read by number, and the gradient that goes back to them.
//
// Forward: out[t] = scale * row[id[t]].  Bound by the memory: one 16-byte piece of a row per thread and load (40,001 bf16 rows of 768 out of
// a million: 21 us, 5.7 TB/s read and written; 16 rows: 14 us a call, the launch).
//
// Backward: sums over the t that read a row, in the order of t, without float atomics (two calls give the same bits).  The (id, t) pairs are
// sorted by id -- stable, so t ascends within an id --, the sorted list is cut into runs of 16 or 64 entries, a workgroup sums each run: an id
// whose entries all lie in one run is written at once, the others leave a partial row at the run's head (the id began earlier) or tail
// (it goes on), and a second kernel adds those up from the run where the id begins.  An id read n times costs n / 64 serial steps, not n.
// Bound by the memory too: 131,072 bf16 gradients of 768 into 262,144 rows, a tenth of the reads going to 26 of them: zeros 53 us (7.6 TB/s), sort
// 62, sums 101 (2 TB/s: rows in the order of the ids), join 12.
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
// eight values as they lie in memory
template <int SC>
__device__ __forceinline__ void unpack8(const uint4* raw, float (&v)[8]) {
    if constexpr (SC == SC_F32) {
        const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = __uint_as_float(w[r]);
    } else {
        const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
        for (int r = 0; r < 4; ++r) v[2 * r] = from_half<SC == SC_BF16>((uint16_t)w[r]), v[2 * r + 1] = from_half<SC == SC_BF16>((uint16_t)(w[r] >> 16));
    }
}
template <int SC>
__device__ __forceinline__ void pack8(const float (&v)[8], uint4* raw) {
    if constexpr (SC == SC_F32) {
        raw[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        raw[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = (uint32_t)to_half<SC == SC_BF16>(v[2 * r]) | (uint32_t)to_half<SC == SC_BF16>(v[2 * r + 1]) << 16;
        raw[0] = make_uint4(w[0], w[1], w[2], w[3]);
    }
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

// Zeros.  Rows that follow each other without a gap are one stretch of memory, filled 16 bytes at a time (a division per piece of a row made
// the fill three times as long); otherwise row by row.
struct ZeroArgs {
    void* out;
    int scalar;
    uint64_t ld;
    uint32_t n, dim;
};
__device__ __forceinline__ void zero_rows(const ZeroArgs& a, uint64_t worker, uint64_t workers) {
    const uint32_t e = a.scalar == SC_F32 ? 4u : 2u;
    char* p = reinterpret_cast<char*>(a.out);
    if (a.ld == a.dim) {
        const uint64_t bytes = (uint64_t)a.n * a.dim * e, head = ((16u - ((uintptr_t)p & 15u)) & 15u) < bytes ? (16u - ((uintptr_t)p & 15u)) & 15u : bytes;
        const uint64_t lines = (bytes - head) / 16u, tail = head + lines * 16u;
        for (uint64_t x = worker; x < lines; x += workers) reinterpret_cast<uint4*>(p + head)[x] = make_uint4(0u, 0u, 0u, 0u);
        if (worker < head / e) store_scalar(p, a.scalar, worker, 0.f);
        if (worker < (bytes - tail) / e) store_scalar(p + tail, a.scalar, worker, 0.f);
    } else {
        const uint64_t total = (uint64_t)a.n * a.dim;
        for (uint64_t x = worker; x < total; x += workers) {
            const uint32_t t = (uint32_t)(x / a.dim), k = (uint32_t)(x - (uint64_t)t * a.dim);
            store_scalar(a.out, a.scalar, (uint64_t)t * a.ld + k, 0.f);
        }
    }
}
__global__ __launch_bounds__(256) void zero_rows_kernel(ZeroArgs a) { zero_rows(a, (uint64_t)blockIdx.x * 256u + threadIdx.x, (uint64_t)gridDim.x * 256u); }
inline uint32_t zero_blocks(const ZeroArgs& a, uint32_t threads) {  // about four stores of 16 bytes per thread
    const uint64_t per = (uint64_t)threads * 4u * 16u, bytes = (uint64_t)a.n * a.dim * (a.scalar == SC_F32 ? 4u : 2u), blocks = (bytes + per - 1) / per;
    return (uint32_t)(blocks < 1 ? 1 : blocks < 16384 ? blocks : 16384);
}
inline void launch_zero_rows(void* out, int scalar, uint64_t ld, uint32_t n, uint32_t dim, hipStream_t st) {
    const ZeroArgs a = {out, scalar, ld, n, dim};
    hipLaunchKernelGGL(zero_rows_kernel, dim3(zero_blocks(a, 256)), dim3(256), 0, st, a);
}

// ------------------------------------------------------------------------------------------------ stable sort of (id, t) by id
// Least significant digit first, up to 10 bits a pass.  A wave owns `items` consecutive entries (256, more beyond a million): it counts its digits (first kernel), a
// wave per digit turns the counts of all waves into places within the digit (second kernel), and every wave moves its entries there in order
// (third kernel, which sums the digits' totals up by itself; entries of one digit keep their order because the lanes of a wave rank
// themselves by lane number and the waves by position).  Up to kSmallSort entries are sorted by one workgroup in one launch instead.
constexpr uint32_t kMaxDigit = 10, kMaxBins = 1u << kMaxDigit, kBatch = 16, kSmallSort = 4096;

struct SortArgs {
    const void* ids;
    uint32_t id_bytes, n, rows;    // ids beyond the rows sort last as `rows`
    uint32_t first, shift, digit;  // first pass: keys come from ids
    const uint32_t *key_in, *pos_in;
    uint32_t *key_out, *pos_out;
    uint32_t* counts;              // [bins][waves], then [bins] totals
    uint32_t waves, items;
};
__device__ __forceinline__ uint32_t key_of(const void* ids, uint32_t id_bytes, uint32_t rows, uint32_t t) {
    const int64_t id = load_id(ids, id_bytes, t);
    return id >= 0 && id < (int64_t)rows ? (uint32_t)id : rows;
}
__device__ __forceinline__ uint32_t sort_key(const SortArgs& a, uint32_t t) { return a.first ? key_of(a.ids, a.id_bytes, a.rows, t) : a.key_in[t]; }
// lanes (of `on`) whose digit is this lane's
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, uint32_t bits, uint64_t on) {
    uint64_t same = on;
    for (uint32_t b = 0; b < bits; ++b) {
        const uint64_t m = __ballot((digit >> b) & 1u);
        same &= (digit >> b) & 1u ? m : ~m;
    }
    return same;
}
__device__ __forceinline__ uint32_t wave_inclusive(uint32_t v, uint32_t lane) {
    for (uint32_t o = 1; o < 64; o <<= 1) {
        const uint32_t u = __shfl_up(v, o);
        v += lane >= o ? u : 0u;
    }
    return v;
}
__global__ __launch_bounds__(64) void sort_count_kernel(SortArgs a) {
    __shared__ uint32_t bins[kMaxBins];
    const uint32_t lane = threadIdx.x, t0 = blockIdx.x * a.items, t1 = min(a.n, t0 + a.items), nb = 1u << a.digit;
    for (uint32_t b = lane; b < nb; b += 64) bins[b] = 0;
    __syncthreads();
    for (uint32_t t = t0 + lane; t < t1; t += 64) atomicAdd(&bins[(sort_key(a, t) >> a.shift) & (nb - 1)], 1u);  // (whole numbers: the order does not matter)
    __syncthreads();
    for (uint32_t b = lane; b < nb; b += 64) a.counts[(size_t)b * a.waves + blockIdx.x] = bins[b];
}
__global__ __launch_bounds__(256) void sort_places_kernel(SortArgs a) {
    const uint32_t lane = threadIdx.x & 63u, b = blockIdx.x * 4u + (threadIdx.x >> 6), nb = 1u << a.digit;
    if (b >= nb) return;
    uint32_t* c = a.counts + (size_t)b * a.waves;
    uint32_t at = 0;
    for (uint32_t w = 0; w < a.waves; w += 64) {
        const uint32_t v = w + lane < a.waves ? c[w + lane] : 0u, s = wave_inclusive(v, lane);
        if (w + lane < a.waves) c[w + lane] = at + s - v;
        at += __shfl(s, 63);
    }
    if (lane == 0) a.counts[(size_t)nb * a.waves + b] = at;
}
__global__ __launch_bounds__(64) void sort_move_kernel(SortArgs a) {
    __shared__ uint32_t at[kMaxBins];
    const uint32_t lane = threadIdx.x, t0 = blockIdx.x * a.items, t1 = min(a.n, t0 + a.items), nb = 1u << a.digit;
    uint32_t before = 0;
    for (uint32_t b = 0; b < nb; b += 64) {  // (nb: 64 or more)
        const uint32_t v = a.counts[(size_t)nb * a.waves + b + lane], s = wave_inclusive(v, lane);
        at[b + lane] = before + s - v + a.counts[(size_t)(b + lane) * a.waves + blockIdx.x];
        before += __shfl(s, 63);
    }
    __syncthreads();
    for (uint32_t t = t0; t < t1; t += 64) {
        const bool on = t + lane < t1;
        const uint32_t key = on ? sort_key(a, t + lane) : 0u, digit = (key >> a.shift) & (nb - 1);
        const uint64_t same = same_digit(digit, a.digit, __ballot(on));
        const uint32_t rank = mbcnt(same), to = on ? at[digit] + rank : 0u;
        __syncthreads();
        if (on && rank == 0) at[digit] += (uint32_t)__popcll(same);
        __syncthreads();
        if (on) {
            a.key_out[to] = key;
            a.pos_out[to] = a.first ? t + lane : a.pos_in[t + lane];
        }
    }
}
// n <= kSmallSort, one workgroup of 16 waves: the same, with everything in LDS; 4 bits a pass, so that a wave's counts are a lane's.
// A wave owns 256 entries in 4 rounds of 64.
struct SmallSortArgs {
    const void* ids;
    uint32_t id_bytes, n, rows, bits;
    uint32_t *key_out, *pos_out;
    ZeroArgs zero;  // workgroups behind the first fill the output with zeros meanwhile
};
__global__ __launch_bounds__(1024) void small_sort_kernel(SmallSortArgs a) {
    __shared__ uint32_t key[2][kSmallSort], pos[2][kSmallSort / 2 + 16];  // (positions: 16 bits each)
    __shared__ uint32_t count[16][17], base[16];
    if (blockIdx.x) {
        zero_rows(a.zero, (uint64_t)(blockIdx.x - 1) * 1024u + threadIdx.x, (uint64_t)(gridDim.x - 1) * 1024u);
        return;
    }
    const uint32_t lane = threadIdx.x & 63u, w = threadIdx.x >> 6;
    const auto pos16 = [&](int x) { return reinterpret_cast<uint16_t*>(pos[x]); };
    for (uint32_t t = threadIdx.x; t < a.n; t += 1024) {
        key[0][t] = key_of(a.ids, a.id_bytes, a.rows, t);
        pos16(0)[t] = (uint16_t)t;
    }
    int from = 0;
    const uint32_t per = ((a.n + 15u) / 16u + 63u) & ~63u;  // entries of a wave, at most 256
    const uint32_t t0 = min(a.n, w * per), t1 = min(a.n, t0 + per);
    for (uint32_t shift = 0; shift < a.bits; shift += 4, from ^= 1) {
        if (threadIdx.x < 256) count[threadIdx.x >> 4][threadIdx.x & 15u] = 0;
        __syncthreads();
        uint32_t rank[4], dig[4];
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            const uint32_t t = t0 + r * 64u + lane;
            const bool on = t < t1;
            dig[r] = on ? (key[from][t] >> shift) & 15u : 0u;
            const uint64_t same = same_digit(dig[r], 4, __ballot(on));
            rank[r] = 0;
            if (on) rank[r] = count[w][dig[r]] + mbcnt(same);  // (the wave's own counters, one round after the other)
            __builtin_amdgcn_wave_barrier();
            if (on && mbcnt(same) == 0) count[w][dig[r]] += (uint32_t)__popcll(same);
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        if (threadIdx.x < 16) {  // places of a digit's waves, then of the digits
            uint32_t s = 0;
            for (uint32_t x = 0; x < 16; ++x) {
                const uint32_t c = count[x][threadIdx.x];
                count[x][threadIdx.x] = s;
                s += c;
            }
            base[threadIdx.x] = s;
        }
        __syncthreads();
        uint32_t below = 0;
        if (lane < 16)
            for (uint32_t d = 0; d < lane; ++d) below += base[d];
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            const uint32_t t = t0 + r * 64u + lane;
            const uint32_t b = __shfl(below, dig[r]);
            if (t < t1) {
                const uint32_t to = b + count[w][dig[r]] + rank[r];
                key[from ^ 1][to] = key[from][t];
                pos16(from ^ 1)[to] = pos16(from)[t];
            }
        }
        __syncthreads();
    }
    for (uint32_t t = threadIdx.x; t < a.n; t += 1024) a.key_out[t] = key[from][t], a.pos_out[t] = pos16(from)[t];
}

// ------------------------------------------------------------------------------------------------ sums of the runs
struct RunArgs {
    const uint32_t *key, *pos;
    uint32_t n, rows, dim, chunks, run;
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
// A thread owns 8 columns of a run of kBatch * batches entries; the rows of a batch are all asked for before the first is summed.  Short rows:
// several runs per workgroup.
template <int SC>
__global__ __launch_bounds__(256) void run_sums_kernel(RunArgs a, uint32_t runs, uint32_t per_group, uint32_t lanes) {
    const uint32_t sub = threadIdx.x / lanes, run = blockIdx.x * per_group + sub;
    if (sub >= per_group || run >= runs) return;
    const uint32_t first = run * a.run, last = min(a.n, first + a.run);
    const uint32_t before = first ? a.key[first - 1] : ~0u;
    for (uint32_t c = threadIdx.x - sub * lanes; c < a.chunks; c += lanes) {
        const uint32_t k = c * 8u;
        float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        bool began = a.key[first] == before;  // the id at hand started in an earlier run
        for (uint32_t t0 = first; t0 < last; t0 += kBatch) {
            const uint32_t m = min(kBatch, a.n - t0);
            uint32_t key[kBatch + 1], pos[kBatch];
#pragma unroll
            for (uint32_t t = 0; t < kBatch; t += 4) {  // (the lists are laid out in whole batches; what lies behind the last entry is not used)
                const uint4 x = *reinterpret_cast<const uint4*>(a.key + t0 + t), y = *reinterpret_cast<const uint4*>(a.pos + t0 + t);
                key[t] = x.x, key[t + 1] = x.y, key[t + 2] = x.z, key[t + 3] = x.w;
                pos[t] = y.x, pos[t + 1] = y.y, pos[t + 2] = y.z, pos[t + 3] = y.w;
            }
#pragma unroll
            for (uint32_t t = 0; t < kBatch; ++t) {
                if (t >= m) key[t] = ~0u, pos[t] = 0u;
            }
            key[kBatch] = t0 + kBatch < a.n ? a.key[t0 + kBatch] : ~0u;
            const bool ends = t0 + kBatch >= last;
            uint4 raw[kBatch][SC == SC_F32 ? 2 : 1];
            if (a.wide_in && a.dim - k >= 8) {
#pragma unroll
                for (uint32_t t = 0; t < kBatch; ++t) {  // (ids out of range: their rows exist too, and are not summed)
                    const uint64_t at = (uint64_t)pos[t] * a.grad_ld + k;
                    if constexpr (SC == SC_F32) {
                        raw[t][0] = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(a.grad) + at)[0];
                        raw[t][1] = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(a.grad) + at)[1];
                    } else {
                        raw[t][0] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.grad) + at);
                    }
                }
            } else {
#pragma unroll
                for (uint32_t t = 0; t < kBatch; ++t) {
                    float v[8];
                    load8(a.grad, SC, (uint64_t)pos[t] * a.grad_ld + k, a.dim - k, false, v);
                    pack8<SC>(v, raw[t]);
                }
            }
#pragma unroll
            for (uint32_t t = 0; t < kBatch; ++t) {
                if (key[t] < a.rows) {  // (ids out of range sort last)
                    const uint32_t id = key[t];
                    float v[8];
                    unpack8<SC>(raw[t], v);
#pragma unroll
                    for (int r = 0; r < 8; ++r) s[r] += v[r];
                    const bool goes_on = key[t + 1] == id;
                    if (!goes_on || (ends && t + 1 == kBatch)) {
                        if (began || goes_on) {
                            float* to = a.part + ((size_t)run * 2u + (began ? 0u : 1u)) * (a.chunks * 8u) + k;
                            reinterpret_cast<f32x4*>(to)[0] = f32x4{s[0], s[1], s[2], s[3]};
                            reinterpret_cast<f32x4*>(to)[1] = f32x4{s[4], s[5], s[6], s[7]};
                        } else {
                            finish_row(a, id, k, s);
                        }
                        began = false;
#pragma unroll
                        for (int r = 0; r < 8; ++r) s[r] = 0.f;
                    }
                }
            }
        }
    }
}
// The run whose last id began in it and goes on: tail + heads of the following runs.  Groups of `lanes` threads take every per_group-th head,
// sixteen on their way at a time; their sums are added in the groups' order.
constexpr uint32_t kJoinThreads = 256;
__global__ __launch_bounds__(kJoinThreads) void run_join_kernel(RunArgs a, uint32_t per_group, uint32_t lanes) {
    __shared__ f32x4 sums[kJoinThreads][2];
    const uint32_t t1 = (blockIdx.x + 1) * a.run;
    if (t1 >= a.n) return;
    const uint32_t id = a.key[t1 - 1], t0 = blockIdx.x * a.run;
    if (id >= a.rows || a.key[t1] != id) return;
    if (a.key[t0] == id && t0 && a.key[t0 - 1] == id) return;  // it began earlier: that run's workgroup adds up
    // the last run the id reaches into (the keys are sorted)
    uint32_t lo = blockIdx.x + 1, hi = (a.n + a.run - 1) / a.run;
    for (uint32_t s = 1; lo + s < hi; s *= 2) {  // (most reach into the next run only: in growing steps, then by halves)
        if (a.key[(size_t)(lo + s) * a.run] != id) hi = lo + s;
        else lo += s;
    }
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (a.key[(size_t)mid * a.run] == id) lo = mid;
        else hi = mid;
    }
    constexpr uint32_t AHEAD = 16;
    const uint32_t sub = threadIdx.x / lanes, l = threadIdx.x - sub * lanes, w = a.chunks * 8u;
    for (uint32_t c0 = 0; c0 < a.chunks; c0 += lanes) {
        const uint32_t k = (c0 + l) * 8u;
        const bool on = sub < per_group && c0 + l < a.chunks;
        f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
        if (on) {
            for (uint32_t x = blockIdx.x + 1 + sub; x <= lo; x += AHEAD * per_group) {
                f32x4 h[AHEAD][2];
#pragma unroll
                for (uint32_t y = 0; y < AHEAD; ++y) {
                    const float* q = a.part + (size_t)min(x + y * per_group, lo) * 2u * w + k;
                    h[y][0] = reinterpret_cast<const f32x4*>(q)[0], h[y][1] = reinterpret_cast<const f32x4*>(q)[1];
                }
#pragma unroll
                for (uint32_t y = 0; y < AHEAD; ++y)
                    if (x + y * per_group <= lo) s0 += h[y][0], s1 += h[y][1];
            }
        }
        __syncthreads();
        sums[threadIdx.x][0] = s0, sums[threadIdx.x][1] = s1;
        __syncthreads();
        if (on && sub == 0) {
            const float* p = a.part + ((size_t)blockIdx.x * 2u + 1u) * w + k;
            s0 = reinterpret_cast<const f32x4*>(p)[0], s1 = reinterpret_cast<const f32x4*>(p)[1];
            for (uint32_t g = 0; g < per_group; ++g) s0 += sums[g * lanes + l][0], s1 += sums[g * lanes + l][1];
            float s[8] = {s0[0], s0[1], s0[2], s0[3], s1[0], s1[1], s1[2], s1[3]};
            finish_row(a, id, k, s);
        }
    }
}

struct LookupGradLayout {
    size_t key[2], pos[2], counts, part, bytes;
    uint32_t waves, items, run, runs, passes, digit, bits;
    bool small;
};
inline LookupGradLayout lookup_grad_layout(size_t n, size_t rows, size_t dim) {
    LookupGradLayout l = {};
    size_t at = 0;
    const auto take = [&](size_t b) {
        const size_t r = at;
        at += (b + 255) & ~(size_t)255;
        return r;
    };
    l.small = n <= kSmallSort;
    l.items = (uint32_t)std::max<size_t>(256, ((n + 4095) / 4096 + 63) / 64 * 64);
    l.waves = (uint32_t)((n + l.items - 1) / l.items);
    // short runs keep few ids and short rows spread over the chip (a run is summed one entry after the other); long ones, once they fill it by
    // themselves (65,536 threads), leave fewer sums to be joined.  In runs of 16 / 64, us: 14,569 ids x 128 53 / 75, 60,000 x 256 71 / 80,
    // 131,072 x 128 109 / 112; 30,011 x 1536 99 / 88, 131,072 x 768 246 / 229
    l.run = n * ((dim + 7) / 8) < ((size_t)4 << 20) ? kBatch : 4 * kBatch;
    l.runs = (uint32_t)((n + l.run - 1) / l.run);
    l.bits = 1;
    while (l.bits < 31 && (rows >> l.bits)) ++l.bits;  // keys 0 .. rows
    l.passes = (l.bits + kMaxDigit - 1) / kMaxDigit;
    l.digit = (l.bits + l.passes - 1) / l.passes;
    if (l.digit < 6) l.digit = 6;  // (a wave looks at 64 digits at a time)
    for (int x = 0; x < (l.small ? 1 : 2); ++x) l.key[x] = take((size_t)l.runs * l.run * 4), l.pos[x] = take((size_t)l.runs * l.run * 4);
    l.counts = take(l.small ? 0 : ((size_t)l.waves + 1) * (1u << l.digit) * 4);
    l.part = take((size_t)l.runs * 2 * ((dim + 7) / 8 * 8) * 4);
    l.bytes = at;
    return l;
}
inline void launch_lookup_grad(const void* grad, int grad_scalar, uint64_t grad_ld, const void* ids, uint32_t id_bytes, uint32_t n, uint32_t rows, uint32_t dim, float scale,
                               bool accumulate, void* out, int out_scalar, uint64_t out_ld, const LookupGradLayout& l, char* work, hipStream_t st) {
    const uint32_t chunks = (dim + 7) / 8;
    if (!accumulate && !(l.small && n)) launch_zero_rows(out, out_scalar, out_ld, rows, dim, st);
    if (!n) return;
    uint32_t to = 0;
    if (l.small) {
        SmallSortArgs s = {ids, id_bytes, n, rows, l.bits, (uint32_t*)(work + l.key[0]), (uint32_t*)(work + l.pos[0]), {out, out_scalar, out_ld, rows, dim}};
        hipLaunchKernelGGL(small_sort_kernel, dim3(accumulate ? 1u : 1u + std::min(4096u, zero_blocks(s.zero, 1024))), dim3(1024), 0, st, s);
    } else {
        SortArgs s = {};
        s.ids = ids;
        s.id_bytes = id_bytes;
        s.n = n;
        s.rows = rows;
        s.counts = (uint32_t*)(work + l.counts);
        s.waves = l.waves;
        s.items = l.items;
        s.digit = l.digit;
        for (uint32_t pass = 0; pass < l.passes; ++pass, to ^= 1u) {
            s.first = pass == 0;
            s.shift = pass * l.digit;
            s.key_in = (const uint32_t*)(work + l.key[to ^ 1u]), s.pos_in = (const uint32_t*)(work + l.pos[to ^ 1u]);
            s.key_out = (uint32_t*)(work + l.key[to]), s.pos_out = (uint32_t*)(work + l.pos[to]);
            hipLaunchKernelGGL(sort_count_kernel, dim3(l.waves), dim3(64), 0, st, s);
            hipLaunchKernelGGL(sort_places_kernel, dim3((1u << l.digit) / 4), dim3(256), 0, st, s);
            hipLaunchKernelGGL(sort_move_kernel, dim3(l.waves), dim3(64), 0, st, s);
        }
        to ^= 1u;
    }
    RunArgs r = {};
    r.key = (const uint32_t*)(work + l.key[to]), r.pos = (const uint32_t*)(work + l.pos[to]);
    r.n = n, r.rows = rows, r.dim = dim, r.chunks = chunks, r.run = l.run;
    r.grad = grad, r.grad_scalar = grad_scalar, r.grad_ld = grad_ld;
    r.scale = scale;
    r.accumulate = accumulate;
    r.out = out, r.out_scalar = out_scalar, r.out_ld = out_ld;
    r.part = (float*)(work + l.part);
    r.wide_in = wide_rows(grad, grad_scalar, grad_ld), r.wide_out = wide_rows(out, out_scalar, out_ld);
    // rows of up to 32 pieces share a workgroup of one wave, longer ones take 128 or 256 threads each
    const uint32_t threads = chunks <= 64 ? 64 : chunks <= 128 ? 128 : 256, lanes = std::min(chunks, threads), group = threads / lanes;
    const dim3 grid((l.runs + group - 1) / group);
    switch (grad_scalar) {
        case SC_F32: hipLaunchKernelGGL((run_sums_kernel<SC_F32>), grid, dim3(threads), 0, st, r, l.runs, group, lanes); break;
        case SC_F16: hipLaunchKernelGGL((run_sums_kernel<SC_F16>), grid, dim3(threads), 0, st, r, l.runs, group, lanes); break;
        default: hipLaunchKernelGGL((run_sums_kernel<SC_BF16>), grid, dim3(threads), 0, st, r, l.runs, group, lanes); break;
    }
    const uint32_t jl = std::min(chunks, kJoinThreads);
    if (l.runs > 1) hipLaunchKernelGGL(run_join_kernel, dim3(l.runs - 1), dim3(kJoinThreads), 0, st, r, kJoinThreads / jl, jl);
}

}  // namespace learn
}  // namespace vs
