// e4m3 codes with one f32 scale for a block of 128 values (irodori_op_block_norm, irodori_op_block_quantize):
// s = max(amax / 448, 2^-126), codes rne(v / s).  amax is over the finite values: an infinity or a NaN becomes e4m3's
// NaN and its neighbours keep theirs.
#pragma once

#include "common.hpp"

namespace irodori {

constexpr int kBlock = 128;  // columns that share a scale
inline __host__ __device__ int blocks_of(int dim) { return (dim + kBlock - 1) / kBlock; }

// A value from the lane that a DPP control names, within a row of 16 lanes.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, false));
}
// Max over each row of 16 lanes (NaNs are passed over).
__device__ __forceinline__ float row16_max(float v) {
    v = fmaxf(v, dpp<0x128>(v));  // row_ror:8
    v = fmaxf(v, dpp<0x124>(v));  // row_ror:4
    v = fmaxf(v, dpp<0x4E>(v));   // quad_perm [2,3,0,1]
    return fmaxf(v, dpp<0xB1>(v));  // quad_perm [1,0,3,2]
}

template <int N>
__device__ __forceinline__ float abs_max(const float (&v)[N]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) m = fmaxf(m, fabsf(v[i]));
    return m;
}
template <int N>
__device__ __forceinline__ float finite_abs_max(const float (&v)[N]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) m = fabsf(v[i]) < __builtin_inff() ? fmaxf(m, fabsf(v[i])) : m;
    return m;
}
__device__ __forceinline__ float scale_of(float amax) { return fmaxf(__fdiv_rn(amax, 448.f), 1.1754943508222875e-38f); }

// The codes of 8 values: the correctly rounded quotients v / s (the product with the rounded reciprocal, corrected once by
// its exact remainder), rounded to nearest even by the converter.  An infinity's remainder is a NaN.  Remainders of quotients down to the least
// midpoint, 2^-10, have bits down to 2^-56 s, which f32 holds from s = 2^-93 on: below 2^-64 values and scale are multiplied by 2^64 first,
// which is exact.
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float s) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = v[i];
    if (__builtin_expect(s < 0x1p-64f, false)) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] *= 0x1p64f;
        s *= 0x1p64f;
    }
    const float inv = __fdiv_rn(1.f, s);
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float q0 = x[i] * inv;
        q[i] = fmaf(fmaf(-q0, s, x[i]), inv, q0);
    }
    return make_uint2(pack_e4m3(q[0], q[1], q[2], q[3]), pack_e4m3(q[4], q[5], q[6], q[7]));
}
// The first n (>= 1) of 8 codes, to an address of any alignment.
typedef unsigned u32x2_b __attribute__((ext_vector_type(2), aligned(1)));
__device__ __forceinline__ void store_codes8(uint8_t* p, int n, uint2 c) {
    if (n >= 8) {
        u32x2_b o = {c.x, c.y};
        *reinterpret_cast<u32x2_b*>(p) = o;
    } else {
#pragma unroll
        for (int i = 0; i < 7; i++)
            if (i < n) p[i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
    }
}

// 8 elements at an address aligned to the element, as they lie in memory (those from n on are zero): no conversion, so that
// many loads go out before the first is waited for.
template <typename T>
struct Raw8 {
    T v __attribute__((ext_vector_type(8)));
};
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T* p, int n) {
    typedef T V __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < 8; i++) r.v[i] = static_cast<T>(0.f);
    if (n >= 8) {
        r.v = *reinterpret_cast<const V*>(p);
    } else if (n > 0) {
#pragma unroll
        for (int i = 0; i < 7; i++)
            if (i < n) r.v[i] = p[i];
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void to_f32x8(const Raw8<T>& r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = static_cast<float>(r.v[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const float (&f)[8]) {
    typedef T V __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    if (n >= 8) {
        V o;
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = static_cast<T>(f[i]);
        *reinterpret_cast<V*>(p) = o;
    } else {
#pragma unroll
        for (int i = 0; i < 7; i++)
            if (i < n) p[i] = static_cast<T>(f[i]);
    }
}

}  // namespace irodori
