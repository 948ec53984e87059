// layers.h -- device building blocks of the operators around RACE attention
// (rms_norm.hip, block_fp8.hip, adamw.hip): rows in vectors of any alignment, sums
// over lanes, and 8-bit blocks.
//
// 8-bit blocks: e4m3 codes with one power-of-two scale 2^s for a block, s the least
// with amax / 2^s <= 448 (e4m3's largest), stored as the byte s + 127 (e8m0).  A power
// of two divides exactly, so a code is the value rounded once, whoever computes it,
// and the matrix cores apply such scales themselves (v_mfma_scale_f32_*).  A scale of
// amax / 448 would use at most one more binade of e4m3's 18, and no more of its 4
// significant bits.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace race {

typedef __bf16 bf16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int BLK = 128;  // elements of an 8-bit block along a row

// ------------------------------------------------------------ vectors of any alignment
// memcpy of 8 to 32 bytes: global loads and stores of up to 16 bytes take any address.
template <typename T, int V> __device__ __forceinline__ void ld_vec(const T *p, float (&r)[V]) {
    T t[V];
    __builtin_memcpy(t, p, sizeof t);
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = (float)t[j];
}
template <typename T, int V> __device__ __forceinline__ void st_vec(T *p, const float (&r)[V]) {
    T t[V];
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = (T)r[j];
    __builtin_memcpy(p, t, sizeof t);
}
// elements c .. c+V-1 of a row of n: zeros behind its end
template <typename T, int V> __device__ __forceinline__ void ld_row(const T *row, int64_t c, int64_t n, float (&r)[V]) {
    if (c + V <= n) {
        ld_vec<T, V>(row + c, r);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = c + j < n ? (float)row[c + j] : 0.f;
    }
}
template <typename T, int V> __device__ __forceinline__ void st_row(T *row, int64_t c, int64_t n, const float (&r)[V]) {
    if (c + V <= n) {
        st_vec<T, V>(row + c, r);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j < n) row[c + j] = (T)r[j];
    }
}

// ------------------------------------------------------------ lanes
template <int CTRL> __device__ __forceinline__ float dpp_move(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// f over the 16 lanes of a row, in every lane of it
template <typename F> __device__ __forceinline__ float row16(float x, F f) {
    x = f(x, dpp_move<0xB1>(x));   // quad_perm [1,0,3,2]
    x = f(x, dpp_move<0x4E>(x));   // quad_perm [2,3,0,1]
    x = f(x, dpp_move<0x141>(x));  // row_half_mirror
    return f(x, dpp_move<0x140>(x));  // row_mirror
}
struct Add { __device__ float operator()(float a, float b) const { return a + b; } };
struct Max { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
// over n = 16, 32 or 64 neighbouring lanes
template <int N, typename F> __device__ __forceinline__ float lanes(float x, F f) {
    x = row16(x, f);
    if constexpr (N >= 32) x = f(x, __shfl_xor(x, 16, 64));
    if constexpr (N >= 64) x = f(x, __shfl_xor(x, 32, 64));
    return x;
}

// ------------------------------------------------------------ 8-bit blocks
// |x| of a finite x, 0 otherwise: infinities and NaN become NaN codes and leave the
// scale of their block to its other elements
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < __builtin_inff() ? a : 0.f;
}
// the scale byte s + 127: amax = f 2^(E-127), 448 = 1.75 * 2^8
__device__ __forceinline__ int scale_byte(float amax) {
    const uint32_t u = __builtin_bit_cast(uint32_t, amax);
    const int b = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);
    return u == 0 ? 127 : b < 0 ? 0 : b;
}
// 2^-s of a scale byte (at most 247), and 2^s
__device__ __forceinline__ float inv_scale(int b) { return __builtin_bit_cast(float, (uint32_t)(254 - b) << 23); }
__device__ __forceinline__ float scale_of(int b) { return __builtin_bit_cast(float, b ? (uint32_t)b << 23 : 1u << 22); }

// four codes, round to nearest even (the instruction returns NaN for what is not finite)
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
// codes c .. c+V-1 of a row whose V divides 128: all of them up to the row's end
template <int V>
__device__ __forceinline__ void st_codes(uint8_t *row, int64_t c, int64_t n, const float (&y)[V], float inv) {
    uint32_t q[V / 4];
#pragma unroll
    for (int j = 0; j < V / 4; ++j)
        q[j] = codes4(y[4 * j] * inv, y[4 * j + 1] * inv, y[4 * j + 2] * inv, y[4 * j + 3] * inv);
    if (c + V <= n) {
        __builtin_memcpy(row + c, q, V);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j < n) row[c + j] = (uint8_t)(q[j / 4] >> (8 * (j & 3)));
    }
}

}  // namespace race
