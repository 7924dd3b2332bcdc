// learn_device.hpp -- scalar helpers of the learning operators' kernels (learn.hip, learn_product.hpp).
#pragma once
#include "hnsw_device.hpp"

namespace vs {
namespace learn {

using f32x4 = __attribute__((ext_vector_type(4))) float;

constexpr float kLog2e = 1.44269504088896340736f, kLog2eLo = 1.9259629911266175e-8f,  // log2(e) = their sum
                kLn2 = 0.693147180559945309417f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }  // one instruction; below 2^-126 it returns 0: such a term is nothing beside the 1 of the row's maximum

template <bool BF16>
__device__ __forceinline__ uint16_t to_half(float f) {
    if constexpr (BF16) return __builtin_bit_cast(uint16_t, (__bf16)f);
    else return __builtin_bit_cast(uint16_t, (_Float16)f);
}
template <bool BF16>
__device__ __forceinline__ float from_half(uint16_t h) {
    if constexpr (BF16) return bf16_bits_to_float(h);
    else return (float)__builtin_bit_cast(_Float16, h);
}

// two (maximum, sum of 2^(z - maximum)) of disjoint column sets
__device__ __forceinline__ float2 join_sums(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    if (m == -__builtin_inff()) return make_float2(m, a.y + b.y);  // nothing yet (or only NaN sums: they stay)
    return make_float2(m, a.y * exp2_fast(a.x - m) + b.y * exp2_fast(b.x - m));
}

// a and b hold one value per lane of two rows of blocks; N = 32: the halves of the wave are joined, lanes 0..31 end up with a's sums and lanes
// 32..63 with b's; N = 16: the same for the odd and even sixteens (a in rows 0 and 2, b in rows 1 and 3)
template <int N>
__device__ __forceinline__ float2 join_swapped(float2 a, float2 b) {
    using u2 = __attribute__((ext_vector_type(2))) unsigned int;
    const auto swap = [](float x, float y) {
        if constexpr (N == 32) return __builtin_bit_cast(u2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false));
        else return __builtin_bit_cast(u2, __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false));
    };
    const u2 m = swap(a.x, b.x), s = swap(a.y, b.y);
    return join_sums(make_float2(__uint_as_float(m[0]), __uint_as_float(s[0])), make_float2(__uint_as_float(m[1]), __uint_as_float(s[1])));
}

__device__ __forceinline__ float load_scalar(const void* p, int scalar, uint64_t i) {
    if (scalar == SC_F32) return reinterpret_cast<const float*>(p)[i];
    const uint16_t h = reinterpret_cast<const uint16_t*>(p)[i];
    return scalar == SC_F16 ? from_half<false>(h) : from_half<true>(h);
}
__device__ __forceinline__ void store_scalar(void* p, int scalar, uint64_t i, float v) {
    if (scalar == SC_F32) reinterpret_cast<float*>(p)[i] = v;
    else reinterpret_cast<uint16_t*>(p)[i] = scalar == SC_F16 ? to_half<false>(v) : to_half<true>(v);
}
__device__ __forceinline__ ushort4 to_half4(int scalar, f32x4 v) {
    ushort4 o;
    if (scalar == SC_F16) o.x = to_half<false>(v[0]), o.y = to_half<false>(v[1]), o.z = to_half<false>(v[2]), o.w = to_half<false>(v[3]);
    else o.x = to_half<true>(v[0]), o.y = to_half<true>(v[1]), o.z = to_half<true>(v[2]), o.w = to_half<true>(v[3]);
    return o;
}
// up to four consecutive elements (`left` of them exist), one wide store where the address allows it
__device__ __forceinline__ void store4(void* p, int scalar, uint64_t i, f32x4 v, uint32_t left) {
    if (scalar == SC_F32) {
        float* to = reinterpret_cast<float*>(p) + i;
        if (left >= 4 && ((uintptr_t)to & 15u) == 0) {
            *reinterpret_cast<f32x4*>(to) = v;
            return;
        }
    } else {
        uint16_t* to = reinterpret_cast<uint16_t*>(p) + i;
        if (left >= 4 && ((uintptr_t)to & 7u) == 0) {
            *reinterpret_cast<ushort4*>(to) = to_half4(scalar, v);
            return;
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if ((uint32_t)r < left) store_scalar(p, scalar, i + r, v[r]);
}

__device__ __forceinline__ f32x4 load4(const void* p, int scalar, uint64_t i, uint32_t left) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (scalar == SC_F32) {
        const float* from = reinterpret_cast<const float*>(p) + i;
        if (left >= 4 && ((uintptr_t)from & 15u) == 0) return *reinterpret_cast<const f32x4*>(from);
    } else {
        const uint16_t* from = reinterpret_cast<const uint16_t*>(p) + i;
        if (left >= 4 && ((uintptr_t)from & 7u) == 0) {
            const ushort4 o = *reinterpret_cast<const ushort4*>(from);
            if (scalar == SC_F16) v = f32x4{from_half<false>(o.x), from_half<false>(o.y), from_half<false>(o.z), from_half<false>(o.w)};
            else v = f32x4{from_half<true>(o.x), from_half<true>(o.y), from_half<true>(o.z), from_half<true>(o.w)};
            return v;
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if ((uint32_t)r < left) v[r] = load_scalar(p, scalar, i + r);
    return v;
}

__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

}  // namespace learn
}  // namespace vs
