// Device code that the attention kernels over the caches share (kernels_kv4.hip,
// kernels_paged_attn.hip): rows, the two f16 terms of a value, sums over a query row's lanes.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vx {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}

__device__ __forceinline__ h8 join8(const h2 *c) {
    return __builtin_shufflevector(__builtin_shufflevector(c[0], c[1], 0, 1, 2, 3),
                                   __builtin_shufflevector(c[2], c[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

// Eight values of a row.
__device__ __forceinline__ void load8(const float *p, bool vec, float *x) {
    if (vec) {
        const f4 a = *reinterpret_cast<const f4 *>(p), b = *reinterpret_cast<const f4 *>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
}

// Weights are taken as 2^(s - m), of a score s and the row's reference m. m moves to kRaise below
// a score that exceeds it by more than kMost: a weight is then at most 2^15, within f16, and the
// largest score's at least about 2^kRaise, so that the low f16 terms of lesser ones stay normal.
constexpr float kMost = 15.0f, kRaise = 7.0f;

__device__ __forceinline__ f4 mfma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Over the four lanes l, l + 16, l + 32, l + 48 that share a query row: v_permlane16_swap
// and v_permlane32_swap put both partners' values into every lane.
__device__ __forceinline__ float row_max(float v) {
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
    u = __builtin_bit_cast(uint32_t, v);
    const auto t = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)t[0]), __builtin_bit_cast(float, (uint32_t)t[1]));
}
__device__ __forceinline__ float row_sum(float v) {
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
    u = __builtin_bit_cast(uint32_t, v);
    const auto t = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (uint32_t)t[0]) + __builtin_bit_cast(float, (uint32_t)t[1]);
}

// A row's scale: below 2^10, the low f16 term of a value down to 2^-13 of the row's largest
// is still normal. The exponent of its largest magnitude; 0 where that is 0 or not finite.
__device__ __forceinline__ int scale_of(float top) {
    return top > 0.f && top < INFINITY ? max(__builtin_amdgcn_frexp_expf(top), -100) : 0;
}
// Eight values times `up`, rounded to f32, as two f16 terms. The compiler must not see that v is a
// product: it makes hi of it once in one rounding (v_fma_mixlo_f16) and once in two, and where
// those differ, one value in 2^13, the low term belongs to another high one.
__device__ __forceinline__ void split8(const float *x, float up, h8 &hi, h8 &lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float v = x[i] * up;
        asm("" : "+v"(v));
        hi[i] = (_Float16)v;
        lo[i] = (_Float16)(v - (float)hi[i]);
    }
}
// Eight weights as two f16 terms; `minus` is -1 that the compiler cannot see, so that v - hi
// is one v_fma_mix_f32.
__device__ __forceinline__ void two_terms(const float *v, float minus, h8 &hi, h8 &lo) {
    h2 h[4], r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        h[e] = __builtin_convertvector((f2{v[2 * e], v[2 * e + 1]}), h2);
        r[e] = __builtin_convertvector((f2{__builtin_fmaf(minus, (float)h[e][0], v[2 * e]),
                                           __builtin_fmaf(minus, (float)h[e][1], v[2 * e + 1])}), h2);
    }
    hi = join8(h);
    lo = join8(r);
}

}  // namespace
}  // namespace vx
