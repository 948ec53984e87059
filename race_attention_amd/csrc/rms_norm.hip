// rms_norm.hip -- gfx950 kernels of the root-mean-square norm with the residual's
// addition, its backward pass, and its output in 8-bit blocks.
//
//   h = x + residual,  rstd = 1 / sqrt(mean(h^2) + eps),  y = h rstd w
//   g = dy w,  dh = rstd (g - h rstd^2 mean(g h)) + dh_out,  dx = dresidual = dh,
//   dw = sum over rows of dy h rstd
//
// h is rounded once, to the residual's type, where it is stored; y normalises the
// unrounded sum.  The backward forms the same sum from x and the residual, or reads h
// where it is fp32 (a bf16 h is 2^-9 off, which dw, a long fp32 sum, would show).
//
// Bound by memory: every array is read or written once.  A row is held in registers by
// one wave (up to 1024 columns, four rows a workgroup, so that no barrier is needed and
// a decode batch of a few rows still starts as many workgroups) or by a workgroup of
// 256 threads (up to 16384 columns, 4096 to codes); longer rows are read twice.  Vectors start at
// any address (an odd row length shifts every row).
#include "layers.h"

namespace race {

struct NormArgs {
    const void *x, *r, *dy, *dh;
    const float *w;
    const float *rstd_in;
    void *y, *h, *dx, *dr;
    uint8_t *scale;
    float *rstd, *dw_part;
    int64_t rows, D;
    int64_t xs, rs, ys, hs, dys, dhs, dxs, drs, ss;  // row strides, elements
    float eps;
};

constexpr int NORM_THREADS = 256;

// Sum over the L threads of a row (L = 64: a wave; 256: the workgroup).
template <int L> __device__ __forceinline__ float row_total(float x, float *part) {
    x = lanes<64>(x, Add{});
    if constexpr (L > 64) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) part[w] = x;
        __syncthreads();
        x = (part[0] + part[1]) + (part[2] + part[3]);
        __syncthreads();
    }
    return x;
}

// 1 / sqrt(total / D + eps) as a float and what it is short of: the fp32 root, and a step of
// Newton's in 64 bits.
__device__ __forceinline__ float row_rstd(float total, double inv_d, float eps, float &low) {
    const double m = (double)total * inv_d + (double)eps;
    const float r = 1.f / sqrtf((float)m);
    const bool number = r > 0.f && r < __builtin_huge_valf();
    const double d = number ? (double)r * (1.5 - 0.5 * m * (double)r * (double)r) : (double)r;
    low = number ? (float)(d - (double)(float)d) : 0.f;
    return (float)d;
}

// v = v rstd w with one rounding.
template <int V>
__device__ __forceinline__ void scale_once(float (&v)[V], float rstd, float low, const float (&w)[V]) {
    float y[V], sum = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float p = v[j] * rstd, e = __builtin_fmaf(v[j], low, __builtin_fmaf(v[j], rstd, -p));
        y[j] = __builtin_fmaf(p, w[j], e * w[j]);
        sum += y[j];
    }
    if (!no_lane(sum != sum)) {  // infinite weights or roots, where e w is no number: the products as they are
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] = y[j] == y[j] ? y[j] : v[j] * rstd * w[j];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = y[j];
}

// L threads a row, NV vectors of V elements each; NV = 0: any row length, read twice.
// CODES: y in 8-bit blocks of 128 columns.
// Where y's roundings show (fp32, and codes, of which those near a tie change), it takes one: three (the
// root's, shared by the row, and two products') are 5.3e-8 of the norm off, one 3.4e-8, for 3% of the time
// of 8192 x 4096 (43.3 and 45.4 us).  Rounding to bf16, 1.7e-3, hides them.
// bf16 with a residual 65536 x 768: 83 us, 4.9 TB/s; to codes 8192 x 4096: 47 us, 5.0 TB/s (a large copy: 5.1).
template <typename TX, typename TR, int V, int NV, int L, bool CODES>
__global__ __launch_bounds__(NORM_THREADS) void k_rms_norm(NormArgs a) {
    constexpr int RPB = NORM_THREADS / L;
    constexpr bool ONCE = CODES || std::is_same<TX, float>::value;
    __shared__ float part[4];
    const int t = threadIdx.x % L;
    const double inv_d = 1. / (double)a.D;
    const int nv = NV ? NV : (int)((a.D + V * L - 1) / (V * L));
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / L; row < a.rows; row += (int64_t)gridDim.x * RPB) {
        const TX *x = (const TX *)a.x + row * a.xs;
        const TR *r = a.r ? (const TR *)a.r + row * a.rs : nullptr;
        auto load = [&](int i, float(&v)[V]) {
            const int64_t c = ((int64_t)i * L + t) * V;
            ld_row<TX, V>(x, c, a.D, v);
            if (r) {
                float u[V];
                ld_row<TR, V>(r, c, a.D, u);
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] += u[j];
            }
        };
        float v[NV ? NV : 1][V], sq = 0.f;
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) load(i, v[i]);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) sq += v[i][j] * v[i][j];
        } else {
            for (int i = 0; i < nv; ++i) {
                load(i, v[0]);
#pragma unroll
                for (int j = 0; j < V; ++j) sq += v[0][j] * v[0][j];
            }
        }
        const float total = row_total<L>(sq, part);
        float rstd, low = 0.f;
        if constexpr (ONCE) rstd = row_rstd(total, inv_d, a.eps, low);
        else rstd = 1.f / sqrtf(total * (float)inv_d + a.eps);
        if (a.rstd && t == 0) a.rstd[row] = rstd;
        auto store = [&](int i, float(&v)[V]) {
            const int64_t c = ((int64_t)i * L + t) * V;
            if (no_lane(c < a.D)) return;
            if (r) st_row<TR, V>((TR *)a.h + row * a.hs, c, a.D, v);
            float w[V];
            ld_row<float, V>(a.w, c, a.D, w);
            if constexpr (ONCE) {
                scale_once<V>(v, rstd, low, w);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = v[j] * rstd * w[j];
            }
            if constexpr (CODES) {
                float amax = 0.f;  // (NaN are left out by fmaxf)
#pragma unroll
                for (int j = 0; j < V; ++j) amax = fmaxf(amax, fabsf(v[j]));
                if (!no_lane(amax == __builtin_huge_valf())) {
                    amax = 0.f;
#pragma unroll
                    for (int j = 0; j < V; ++j) amax = fmaxf(amax, finite_abs(v[j]));
                }
                const int b = scale_byte(lanes<BLK / V>(amax, Max{}));
                st_codes<V>((uint8_t *)a.y + row * a.ys, c, a.D, v, scale_of(b));
                if (c % BLK == 0 && c < a.D) a.scale[row * a.ss + c / BLK] = (uint8_t)b;
            } else {
                st_row<TX, V>((TX *)a.y + row * a.ys, c, a.D, v);
            }
        };
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) store(i, v[i]);
        } else {
            for (int i = 0; i < nv; ++i) {
                load(i, v[0]);
                store(i, v[0]);
            }
        }
    }
}

// Backward.  A workgroup walks rows and keeps its part of dw in registers (NV = 0: in
// its row of dw_part): dw_part[workgroup][D], added by k_column_sum in a fixed order.
// The sum is x + r, or r alone where x is NULL.
// A row is a chain of loads, a sum over its lanes and stores; AHEAD (rows of few registers): the next
// row's loads are on their way meanwhile, and w stays in registers (8192 x 4096 bf16 with a residual:
// 85 us without, 67 with).  bf16 waits in pairs: as single values it took a register each, and 65536 x
// 768 with a residual 163 us; it takes 88 (dx past the caches; 105 through them).
template <typename TX, typename TR, int V, int NV, int L>
__global__ __launch_bounds__(NORM_THREADS) void k_rms_norm_bwd(NormArgs a) {
    constexpr int RPB = NORM_THREADS / L, N = NV ? NV : 1;
    constexpr bool AHEAD = NV > 0 && NV * V <= 16;
    __shared__ float part[4];
    const int t = threadIdx.x % L;
    const float inv_d = 1.f / (float)a.D;
    const int nv = NV ? NV : (int)((a.D + V * L - 1) / (V * L));
    auto column = [&](int i) { return ((int64_t)i * L + t) * V; };
    float dw[N][V], wr[AHEAD ? N : 1][V];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) dw[i][j] = 0.f;
    if constexpr (AHEAD) {
#pragma unroll
        for (int i = 0; i < NV; ++i) ld_row<float, V>(a.w, column(i), a.D, wr[i]);
    }
    float *out = a.dw_part + blockIdx.x * a.D;
    if constexpr (NV == 0) {
        for (int64_t c = threadIdx.x; c < a.D; c += NORM_THREADS) out[c] = 0.f;
        __syncthreads();
    }
    struct Vec {  // of a row, as loaded
        Raw<TX, V> x, dy;
        Raw<TR, V> r, dh;
        __device__ __forceinline__ void h(const NormArgs &a, float (&v)[V]) const {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = a.x ? x[j] + r[j] : r[j];
        }
    };
    auto load = [&](int64_t row, int i, Vec &v) {
        const int64_t c = column(i);
        v.r.load((const TR *)a.r + row * a.rs, c, a.D);
        v.dy.load((const TX *)a.dy + row * a.dys, c, a.D);
        if (a.x) v.x.load((const TX *)a.x + row * a.xs, c, a.D);
        if (a.dh) v.dh.load((const TR *)a.dh + row * a.dhs, c, a.D);
    };
    auto weights = [&](int i, float(&w)[V]) {
        if constexpr (AHEAD) {
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = wr[i][j];
        } else {
            ld_row<float, V>(a.w, column(i), a.D, w);
        }
    };
    const int64_t row0 = (int64_t)blockIdx.x * RPB + threadIdx.x / L, stride = (int64_t)gridDim.x * RPB;
    Vec v[N], next[AHEAD ? N : 1];
    if constexpr (AHEAD) {
        if (row0 < a.rows)
#pragma unroll
            for (int i = 0; i < NV; ++i) load(row0, i, next[i]);
    }
    for (int64_t row = row0; row < a.rows; row += stride) {
        const float rstd = a.rstd_in[row];
        float gh = 0.f;
        auto dot = [&](int i, const Vec &v) {
            float w[V], h[V];
            weights(i, w);
            v.h(a, h);
#pragma unroll
            for (int j = 0; j < V; ++j) gh += v.dy[j] * w[j] * h[j];
        };
        if constexpr (AHEAD) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = next[i];
            if (row + stride < a.rows)
#pragma unroll
                for (int i = 0; i < NV; ++i) load(row + stride, i, next[i]);
#pragma unroll
            for (int i = 0; i < NV; ++i) dot(i, v[i]);
        } else if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) load(row, i, v[i]);
#pragma unroll
            for (int i = 0; i < NV; ++i) dot(i, v[i]);
        } else {
            for (int i = 0; i < nv; ++i) {
                load(row, i, v[0]);
                dot(i, v[0]);
            }
        }
        const float k = row_total<L>(gh, part) * inv_d * rstd * rstd;
        auto finish = [&](int i, const Vec &v, float(&acc)[V]) {
            const int64_t c = column(i);
            float w[V], h[V], d[V];
            weights(i, w);
            v.h(a, h);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                acc[j] += v.dy[j] * (h[j] * rstd);
                d[j] = rstd * (v.dy[j] * w[j] - h[j] * k);
            }
            if (a.dh) {
#pragma unroll
                for (int j = 0; j < V; ++j) d[j] += v.dh[j];
            }
            if (a.dx) st_row<TX, V>((TX *)a.dx + row * a.dxs, c, a.D, d);
            if (a.dr) st_row<TR, V>((TR *)a.dr + row * a.drs, c, a.D, d);
        };
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) finish(i, v[i], dw[i]);
        } else {
            for (int i = 0; i < nv; ++i) {
                const int64_t c = column(i);
                load(row, i, v[0]);
                ld_row<float, V>(out, c, a.D, dw[0]);
                finish(i, v[0], dw[0]);
                st_row<float, V>(out, c, a.D, dw[0]);
            }
        }
    }
    if constexpr (NV > 0) {
        if constexpr (RPB > 1) {
            // the four rows' waves: added through LDS, wave by wave
            __shared__ float acc[NV * V * L];
            for (int w = 0; w < RPB; ++w) {
                if (threadIdx.x / L == w) {
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            float &s = acc[(i * V + j) * L + t];
                            s = w ? s + dw[i][j] : dw[i][j];
                        }
                }
                __syncthreads();
            }
            for (int i = 0; i < NV; ++i)
                for (int jr = threadIdx.x / L; jr < V; jr += RPB) {
                    const int64_t c = column(i) + jr;
                    if (c < a.D) out[c] = acc[(i * V + jr) * L + t];
                }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) st_row<float, V>(out, column(i), a.D, dw[i]);
        }
    }
}

// out[c] = sum over p < P of part[p][c], in a fixed order: 16 threads a column take every
// 16th row, and their sums are added in a tree.  (fp32: at most P / 16 terms in a chain.)
constexpr int CS_COLS = 16;
template <typename TO>
__global__ __launch_bounds__(256) void k_column_sum(const float *__restrict__ part, TO *__restrict__ out, int P,
                                                    int64_t C) {
    __shared__ float s[16][CS_COLS + 1];
    const int cl = threadIdx.x % CS_COLS, pr = threadIdx.x / CS_COLS;
    const int64_t c = (int64_t)blockIdx.x * CS_COLS + cl;
    float x = 0.f;
    if (c < C) {
#pragma unroll 8
        for (int p = pr; p < P; p += 16) x += part[(int64_t)p * C + c];
    }
    s[pr][cl] = x;
    __syncthreads();
    for (int n = 8; n > 0; n >>= 1) {
        if (pr < n) s[pr][cl] += s[pr + n][cl];
        __syncthreads();
    }
    if (pr == 0 && c < C) out[c] = (TO)s[0][cl];
}

}  // namespace race
