// adamw.hip -- gfx950 kernels of one AdamW step over many tensors.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p - lr wd p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// with m and v in fp32, or in 8-bit blocks of 128 neighbouring elements: m, and in
// place of v its root.  (e4m3 spans 2^18, so the roots in a block span as much and v
// 2^36.)  8-bit states are rounded stochastically: b2 = 0.999 changes v by a thousandth a
// step, a sixtieth of the distance of neighbouring codes, and rounded to the nearest it
// would never move.  The random numbers are a hash of the seed and the element's place:
// the same call gives the same result.
//
// Bound by memory (28 bytes a parameter, 16 with 8-bit states): one launch takes up to
// ADAM_TENSORS tensors, whose pointers travel as its arguments, and a workgroup a run of
// ADAM_CHUNK elements of one tensor.  162.9 M parameters in 161 tensors (four launches): fp32 states 881 us,
// 5.2 TB/s; 8 bits 513 us, 5.1 TB/s (a large copy: 5.1).  11 M in 83: 71 us, 4.3 TB/s, the ends of two launches.
#include "layers.h"

namespace race {

constexpr int ADAM_TENSORS = 48, ADAM_THREADS = 256, ADAM_CHUNK = 4096;

struct AdamArgs {
    void *p[ADAM_TENSORS];
    const void *g[ADAM_TENSORS];
    void *m[ADAM_TENSORS], *v[ADAM_TENSORS];
    uint8_t *ms[ADAM_TENSORS], *vs[ADAM_TENSORS];
    int64_t n[ADAM_TENSORS];
    uint32_t first[ADAM_TENSORS];  // the tensor's first workgroup
    uint32_t place[ADAM_TENSORS];  // of its first element among the call's, in whole blocks; mod 2^32
    int count;
    uint32_t seed, mixed_seed;     // mixed_seed = mix32(seed); with a device step mix32(seed + step)
    float b1, c1, b2, c2, keep, lr_bc1, inv_root_bc2, eps;  // c = 1 - b, keep = 1 - lr wd
    double lr, db1, db2;
    const float *step;  // nullable: the step on the device, in place of lr_bc1 and inv_root_bc2
};
static_assert(sizeof(AdamArgs) <= 4096, "kernel arguments");

// 32 bits of a 32-bit whole number: two rounds of xor-shift and multiplication
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x7feb352du;
    x = (x ^ (x >> 15)) * 0x846ca68bu;
    return x ^ (x >> 16);
}

// y, |y| <= 448, to a neighbouring e4m3 number: up with the probability of the
// remainder.  Exact in fp32 but for the sum with u, at most 2^-20 of a spacing off.
__device__ __forceinline__ float stochastic(float y, float u) {
    const uint32_t e = (__builtin_bit_cast(uint32_t, y) >> 23) & 255u;
    const uint32_t se = (e < 121u ? 121u : e) - 3u;  // of the spacing: 3 bits behind the leading one, 2^-9 below 2^-6
    const float step = __builtin_bit_cast(float, se << 23), inv = __builtin_bit_cast(float, (254u - se) << 23);
    return __builtin_copysignf(floorf(fabsf(y) * inv + u) * step, y);
}

template <typename TP, typename TG, bool EIGHT> __global__ __launch_bounds__(ADAM_THREADS) void k_adamw(AdamArgs a) {
    constexpr int V = EIGHT ? 8 : 4;
    int t = 0;
    for (int s = 32; s > 0; s >>= 1)
        if (t + s < a.count && a.first[t + s] <= blockIdx.x) t += s;
    const int64_t n = a.n[t], c0 = (int64_t)(blockIdx.x - a.first[t]) * ADAM_CHUNK;
    float lr_bc1 = a.lr_bc1, inv_root_bc2 = a.inv_root_bc2;
    uint32_t mixed_seed = a.mixed_seed;
    if (a.step) {
        const double k = (double)*a.step;
        lr_bc1 = (float)(a.lr / (1.0 - pow(a.db1, k)));
        inv_root_bc2 = (float)(1.0 / sqrt(1.0 - pow(a.db2, k)));
        mixed_seed = mix32(a.seed + (uint32_t)k);
    }
    TP *p = (TP *)a.p[t];
    const TG *g = (const TG *)a.g[t];
    auto update = [&](float(&pv)[V], const float(&gv)[V], float(&mv)[V], float(&vv)[V], float(&root)[V]) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            mv[j] = a.b1 * mv[j] + a.c1 * gv[j];
            vv[j] = a.b2 * vv[j] + a.c2 * gv[j] * gv[j];
            root[j] = sqrtf(vv[j]);
            pv[j] = pv[j] * a.keep - lr_bc1 * mv[j] / (root[j] * inv_root_bc2 + a.eps);
        }
    };
#pragma unroll 2
    for (int i = 0; i < ADAM_CHUNK / (ADAM_THREADS * V); ++i) {
        const int64_t c = c0 + (int64_t)(i * ADAM_THREADS + threadIdx.x) * V;
        float pv[V], gv[V], mv[V], vv[V], root[V];
        if constexpr (!EIGHT) {
            if (c >= n) break;
            float *m = (float *)a.m[t], *v = (float *)a.v[t];
            ld_row<TP, V>(p, c, n, pv);
            ld_row<TG, V>(g, c, n, gv);
            ld_row<float, V>(m, c, n, mv);
            ld_row<float, V>(v, c, n, vv);
            update(pv, gv, mv, vv, root);
            st_row<TP, V>(p, c, n, pv);
            st_row<float, V>(m, c, n, mv);
            st_row<float, V>(v, c, n, vv);
        } else {
            if (c - c % BLK >= n) break;  // whole blocks: 16 lanes
            uint8_t *m = (uint8_t *)a.m[t], *r = (uint8_t *)a.v[t];
            ld_row<TP, V>(p, c, n, pv);
            ld_row<TG, V>(g, c, n, gv);
            const int64_t blk = c / BLK;
            const float sm = scale_of(a.ms[t][blk]), sr = scale_of(a.vs[t][blk]);
            auto values = [&](const uint8_t *x, float s, float(&y)[V]) {
                uint32_t q[2] = {0, 0};
                if (c + V <= n) {
                    __builtin_memcpy(q, x + c, V);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (c + j < n) q[j / 4] |= (uint32_t)x[c + j] << (8 * (j & 3));
                }
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    y[4 * w] = __builtin_amdgcn_cvt_f32_fp8((int)q[w], 0) * s;
                    y[4 * w + 1] = __builtin_amdgcn_cvt_f32_fp8((int)q[w], 1) * s;
                    y[4 * w + 2] = __builtin_amdgcn_cvt_f32_fp8((int)q[w], 2) * s;
                    y[4 * w + 3] = __builtin_amdgcn_cvt_f32_fp8((int)q[w], 3) * s;
                }
            };
            values(m, sm, mv);
            values(r, sr, root);
#pragma unroll
            for (int j = 0; j < V; ++j) vv[j] = root[j] * root[j];
            update(pv, gv, mv, vv, root);
            st_row<TP, V>(p, c, n, pv);
            float am = 0.f, ar = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                am = fmaxf(am, finite_abs(mv[j]));
                ar = fmaxf(ar, finite_abs(root[j]));
            }
            const int bm = scale_byte(row16(am, Max{})), br = scale_byte(row16(ar, Max{}));
            const float im = scale_of(254 - bm), ir = scale_of(254 - br);  // 2^-s (bytes are at most 247)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const uint32_t h = mix32(a.place[t] + (uint32_t)(c + j) + mixed_seed);
                mv[j] = stochastic(mv[j] * im, (float)(h & 0xffffu) * 0x1p-16f);
                root[j] = stochastic(root[j] * ir, (float)(h >> 16) * 0x1p-16f);
            }
            st_codes<V>(m, c, n, mv, 1.f);
            st_codes<V>(r, c, n, root, 1.f);
            if (c % BLK == 0) {
                a.ms[t][blk] = (uint8_t)bm;
                a.vs[t][blk] = (uint8_t)br;
            }
        }
    }
}

}  // namespace race
