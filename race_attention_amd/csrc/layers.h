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
// The bytes of t, 8 or 16, to any address, as data that this launch does not touch again.  The caches then give up
// lines that are read again less often (us: product 50240 x 1536, K = 384, 82 and 69; norm forward and
// backward of 65536 x 768 191 and 173).  Lanes must fill lines together: 32 bytes a lane, in two stores, are
// slower so (fp32 8192 x 16384: 407 and 508), and stay as they were.
template <typename A> __device__ __forceinline__ void st_stream(void *p, const A &t) {
    typedef int words __attribute__((ext_vector_type(sizeof(A) / 4), aligned(1)));
    words w;
    __builtin_memcpy(&w, &t, sizeof w);
    __builtin_nontemporal_store(w, (words *)p);
}
// whether a condition holds in none of the wave's active lanes: a branch on it is the wave's, so its
// other side costs nothing
__device__ __forceinline__ bool no_lane(bool x) { return __builtin_amdgcn_ballot_w64(x) == 0; }
// elements of the row from c on, 0 to V, as a number that the compiler does not form before the
// branch that uses it
template <int V> __device__ __forceinline__ int left_in_row(int64_t c, int64_t n) {
    int left = n - c < V ? (int)(n - c) : V;
    left = left < 0 ? 0 : left;
    asm volatile("" : "+v"(left));
    return left;
}
// elements c .. c+V-1 of a row of n >= 1: zeros behind its end.  (A wave that reaches it loads elements
// one by one, the first again in place of what lies behind it: loads under a condition each would wait
// for each other.)
template <typename T, int V> __device__ __forceinline__ void ld_raw(const T *row, int64_t c, int64_t n, T (&t)[V]) {
    if (no_lane(c + V > n)) {
        __builtin_memcpy(t, row + c, sizeof t);
    } else if (no_lane(c < n)) {
#pragma unroll
        for (int j = 0; j < V; ++j) t[j] = (T)0.f;
    } else {
        const int left = left_in_row<V>(c, n);
        const T *p = row + (left ? c : 0);
#pragma unroll
        for (int j = 0; j < V; ++j) t[j] = p[j < left ? j : 0];
#pragma unroll
        for (int j = 0; j < V; ++j) t[j] = j < left ? t[j] : (T)0.f;
    }
}
// V elements as they were loaded, in whole registers (bf16 in pairs)
template <typename T, int V> struct Raw;
template <int V> struct Raw<float, V> {
    float f[V];
    __device__ __forceinline__ void load(const float *row, int64_t c, int64_t n) { ld_raw<float, V>(row, c, n, f); }
    __device__ __forceinline__ float operator[](int j) const { return f[j]; }
};
template <int V> struct Raw<bf16, V> {
    uint32_t w[V / 2];
    __device__ __forceinline__ void load(const bf16 *row, int64_t c, int64_t n) {
        if (no_lane(c + V > n)) {
            __builtin_memcpy(w, row + c, sizeof w);
        } else if (no_lane(c < n)) {
#pragma unroll
            for (int j = 0; j < V / 2; ++j) w[j] = 0;
        } else {
            const int left = left_in_row<V>(c, n);
            const bf16 *p = row + (left ? c : 0);
            uint16_t t[V];
#pragma unroll
            for (int j = 0; j < V; ++j) __builtin_memcpy(&t[j], p + (j < left ? j : 0), 2);
#pragma unroll
            for (int j = 0; j < V / 2; ++j)
                w[j] = (2 * j < left ? t[2 * j] : 0u) | (uint32_t)(2 * j + 1 < left ? t[2 * j + 1] : 0u) << 16;
        }
    }
    __device__ __forceinline__ float operator[](int j) const {
        return __builtin_bit_cast(float, j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
    }
};
template <typename T, int V> __device__ __forceinline__ void ld_row(const T *row, int64_t c, int64_t n, float (&r)[V]) {
    T t[V];
    ld_raw<T, V>(row, c, n, t);
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = (float)t[j];
}
template <typename T, int V> __device__ __forceinline__ void st_row(T *row, int64_t c, int64_t n, const float (&r)[V]) {
    if (c + V <= n) {
        T t[V];
#pragma unroll
        for (int j = 0; j < V; ++j) t[j] = (T)r[j];
        if constexpr (sizeof t <= 16) st_stream(row + c, t);
        else __builtin_memcpy(row + c, t, sizeof t);
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
// 2^s of a scale byte
__device__ __forceinline__ float scale_of(int b) { return __builtin_bit_cast(float, b ? (uint32_t)b << 23 : 1u << 22); }

// four codes of values divided by scale, a power of two: round to nearest even, NaN for what is
// not finite
typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float scale) {
    i16x2 r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
    return __builtin_bit_cast(uint32_t, r);
}
// of two pairs of bf16
__device__ __forceinline__ uint32_t codes4(uint32_t ab, uint32_t cd, float scale) {
    i16x2 r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, ab), scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, cd), scale, true);
    return __builtin_bit_cast(uint32_t, r);
}
// V codes from column c of a row on, those before column n
template <int V> __device__ __forceinline__ void st_codes(uint8_t *row, int64_t c, int64_t n, const uint32_t (&q)[V / 4]) {
    if (c + V <= n) {
        __builtin_memcpy(row + c, q, V);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j < n) row[c + j] = (uint8_t)(q[j / 4] >> (8 * (j & 3)));
    }
}
template <int V>
__device__ __forceinline__ void st_codes(uint8_t *row, int64_t c, int64_t n, const float (&y)[V], float scale) {
    uint32_t q[V / 4];
#pragma unroll
    for (int j = 0; j < V / 4; ++j) q[j] = codes4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3], scale);
    st_codes<V>(row, c, n, q);
}

// Pairs of bf16 in words: |x| of finite elements (0 for the others) as 16-bit numbers, whose
// order is theirs.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2 abs2(uint32_t w) { return __builtin_bit_cast(u16x2, w & 0x7fff7fffu); }
__device__ __forceinline__ u16x2 finite_abs2(uint32_t w) {
    const i16x2 x = __builtin_bit_cast(i16x2, w & 0x7fff7fffu);
    return __builtin_bit_cast(u16x2, x & ((x - (short)0x7f80) >> 15));
}
__device__ __forceinline__ float larger(u16x2 m) {
    return __builtin_bit_cast(float, (uint32_t)(m[0] > m[1] ? m[0] : m[1]) << 16);
}

}  // namespace race
