// block_fp8.hip -- gfx950 kernels of matrices in 8-bit blocks: the quantiser and the
// product out = a b^T of two of them.
//
// A matrix [rows][cols] in 8-bit blocks: e4m3 codes and a power-of-two scale for each
// block of 128 columns of one row (activations) or of 128 columns of 128 rows
// (weights).  With S_a, S_b the scales' exponents,
//   out[m][n] = sum_kb 2^(S_a[m,kb] + S_b[n,kb]) sum_{k in block kb} a[m,k] b[n,k].
// v_mfma_scale_f32_16x16x128_f8f6f4 contracts 128 codes and takes a scale byte for
// every row of both operands, so one instruction is one block of a 16x16 tile, without
// any work on the vector units.
//
// The 8-bit matrix instructions (of any depth) add their products with few bits: what is
// under 2^-18 of the largest is lost, and sums of 128 random products are 1.7e-5 of
// their norm off.  That is far under half a step of a bf16 result (2^-9), but not of an
// fp32 one, which is asked for where many products are summed (the weights' gradient).  So
// products with an fp32 output turn the codes into bf16 on the way to the matrix cores
// (v_cvt_scalef32_pk_bf16_fp8 applies the scale; both are exact) and use the bf16
// instructions, which sum in fp32 at half the rate.
#include "layers.h"

namespace race {

// ------------------------------------------------------------ quantiser
struct QuantArgs {
    const void *x;
    int64_t rows, cols, ld;
    uint8_t *codes, *scale;      // [rows][cols], nullable
    int64_t codes_ld, scale_ld;
    uint8_t *codes_t, *scale_t;  // of the transpose, [cols][rows], nullable
    int64_t codes_t_ld, scale_t_ld;
    float *sums;                 // [ceil(rows / 128)][cols] column sums of 128 rows, nullable
};

// Elements of 8 columns as the quantisers hold them: bf16 as it is, in pairs, for which
// comparing and converting take an instruction a pair, or fp32.
template <typename T> struct Eight;
template <> struct Eight<bf16> : Raw<bf16, 8> {
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = 0;
    }
    // (what is not finite is larger than all that is: looked for only where it shows)
    __device__ __forceinline__ float amax() const {
        u16x2 m = abs2(w[0]);
#pragma unroll
        for (int j = 1; j < 4; ++j) m = __builtin_elementwise_max(m, abs2(w[j]));
        if (__builtin_expect(m[0] >= 0x7f80 || m[1] >= 0x7f80, 0)) {
            m = finite_abs2(w[0]);
#pragma unroll
            for (int j = 1; j < 4; ++j) m = __builtin_elementwise_max(m, finite_abs2(w[j]));
        }
        return larger(m);
    }
    __device__ __forceinline__ void codes(float scale, uint32_t (&q)[2]) const {
        q[0] = codes4(w[0], w[1], scale);
        q[1] = codes4(w[2], w[3], scale);
    }
    // of column j of four rows
    static __device__ __forceinline__ uint32_t down(const Eight (&v)[8], int r, int j, float scale) {
        const uint32_t pick = j & 1 ? 0x07060302u : 0x05040100u;  // the high or the low halves of two words
        return codes4(__builtin_amdgcn_perm(v[r + 1].w[j / 2], v[r].w[j / 2], pick),
                      __builtin_amdgcn_perm(v[r + 3].w[j / 2], v[r + 2].w[j / 2], pick), scale);
    }
    // amax of each column over 8 rows
    static __device__ __forceinline__ void columns(const Eight (&v)[8], float (&m)[8]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u16x2 x = finite_abs2(v[0].w[j]);
#pragma unroll
            for (int r = 1; r < 8; ++r) x = __builtin_elementwise_max(x, finite_abs2(v[r].w[j]));
            m[2 * j] = __builtin_bit_cast(float, (uint32_t)x[0] << 16);
            m[2 * j + 1] = __builtin_bit_cast(float, (uint32_t)x[1] << 16);
        }
    }
};
template <> struct Eight<float> : Raw<float, 8> {
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = 0.f;
    }
    __device__ __forceinline__ float amax() const {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(f[j]));
        return m;
    }
    __device__ __forceinline__ void codes(float scale, uint32_t (&q)[2]) const {
        q[0] = codes4(f[0], f[1], f[2], f[3], scale);
        q[1] = codes4(f[4], f[5], f[6], f[7], scale);
    }
    static __device__ __forceinline__ uint32_t down(const Eight (&v)[8], int r, int j, float scale) {
        return codes4(v[r].f[j], v[r + 1].f[j], v[r + 2].f[j], v[r + 3].f[j], scale);
    }
    static __device__ __forceinline__ void columns(const Eight (&v)[8], float (&m)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            m[j] = 0.f;
#pragma unroll
            for (int r = 0; r < 8; ++r) m[j] = fmaxf(m[j], finite_abs(v[r].f[j]));
        }
    }
};

// Rows alone: 16 lanes hold a block of 128 columns.  Bound by memory; 16 blocks a
// workgroup, so that a batch of few rows is spread over the chip.  bf16 50240 x 1536: 38 us, 6 TB/s (part of x
// from the last-level cache); 16 x 4096: 2.1 us, where the tiles below take 3.7.
template <typename T> __global__ __launch_bounds__(256) void k_quantize_rows(QuantArgs a) {
    const int64_t nb = (a.cols + BLK - 1) / BLK, total = a.rows * nb, cend = (a.cols + 15) / 16 * 16;
    const int l = threadIdx.x & 15;
    for (int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); i < total; i += (int64_t)gridDim.x * 16) {
        const int64_t row = i / nb, kb = i % nb, c = kb * BLK + 8 * l;
        Eight<T> v;
        v.load((const T *)a.x + row * a.ld, c, a.cols);
        const int b = scale_byte(row16(v.amax(), Max{}));
        uint32_t q[2];
        v.codes(scale_of(b), q);
        st_codes<8>(a.codes + row * a.codes_ld, c, cend, q);
        if (l == 0) a.scale[row * a.scale_ld + kb] = (uint8_t)b;
    }
}

// A 128 x 128 tile, read once, for any of: the row-wise blocks, the blocks of the
// transpose (128 rows of one column), one block of both (BLOCK), and the column sums.
// Thread (i, l) = (tid / 16, tid % 16) holds 8 rows x 8 columns: the amax of a row is
// one over 16 neighbouring lanes, that of a column one over the 8 rows in registers,
// then over the 16 threads above each other through LDS.  Transposed codes leave through
// LDS in rows of 128 bytes: word w (4 rows) of a column stands at w ^ swizzle(column), so
// that neither the 16 columns 8 apart of a write nor a read's pieces of 8 columns meet in a bank.
// Bound by memory: bf16 50240 x 1536 both ways and its sums, from memory, 65 us (4.8 TB/s); a call for each
// of the three would read x three times.  (Codes past the caches: 300 us for a layer's forward and backward that
// takes 290, whose products read them next.)  fp32 1536 x 384 as 128 x 128 blocks both ways: 6.8 us, 36
// workgroups' latency.
template <typename T, bool BLOCK>
__global__ __launch_bounds__(256) void k_quantize_tile(QuantArgs a) {
    __shared__ float red[16][BLK + 4];
    __shared__ __align__(16) uint32_t tr[BLK * 32];
    const int l = threadIdx.x & 15, i = threadIdx.x >> 4;
    const int64_t r0 = (int64_t)blockIdx.y * BLK, c0 = (int64_t)blockIdx.x * BLK;
    const int64_t c = c0 + 8 * l, cend = (a.cols + 15) / 16 * 16;
    Eight<T> v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const int64_t row = r0 + 8 * i + r;
        if (row < a.rows) v[r].load((const T *)a.x + row * a.ld, c, a.cols);
        else v[r].zero();
    }
    int bt[8];  // scale bytes of the transposed blocks of this thread's 8 columns
    int ball = 0;
    if (BLOCK || a.codes_t) {
        float m[8];
        Eight<T>::columns(v, m);
#pragma unroll
        for (int j = 0; j < 8; ++j) red[i][8 * l + j] = m[j];
        __syncthreads();
        if constexpr (BLOCK) {
            float all = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) all = fmaxf(all, red[i][8 * l + k]);
            all = row16(all, Max{});
            if (l == 0) red[i][BLK] = all;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 16; ++k) all = fmaxf(all, red[k][BLK]);
            ball = scale_byte(all);
        } else {
            if (threadIdx.x < BLK) {
                float x = 0.f;
#pragma unroll
                for (int k = 0; k < 16; ++k) x = fmaxf(x, red[k][threadIdx.x]);
                const int b = scale_byte(x);
                red[0][threadIdx.x] = __builtin_bit_cast(float, b);
                if (c0 + threadIdx.x < a.cols) a.scale_t[(c0 + threadIdx.x) * a.scale_t_ld + blockIdx.y] = (uint8_t)b;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 8; ++j) bt[j] = __builtin_bit_cast(int, red[0][8 * l + j]);
        }
    }
    if (a.codes) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int64_t row = r0 + 8 * i + r;
            int b = ball;
            if constexpr (!BLOCK) b = scale_byte(row16(v[r].amax(), Max{}));
            if (row < a.rows) {
                uint32_t q[2];
                v[r].codes(scale_of(b), q);
                st_codes<8>(a.codes + row * a.codes_ld, c, cend, q);
                if (!BLOCK && l == 0) a.scale[row * a.scale_ld + blockIdx.x] = (uint8_t)b;
            }
        }
        if (BLOCK && threadIdx.x == 0) a.scale[blockIdx.y * a.scale_ld + blockIdx.x] = (uint8_t)ball;
    }
    if (a.codes_t) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float scale = scale_of(BLOCK ? ball : bt[j]);
            const int col = 8 * l + j;
            uint2 q;
            q.x = Eight<T>::down(v, 0, j, scale);
            q.y = Eight<T>::down(v, 4, j, scale);
            // 8-byte piece i of 16, swizzled within the row of 128 bytes
            *(uint2 *)&tr[col * 32 + 2 * (i ^ (l & 15))] = q;
        }
        if (BLOCK && threadIdx.x == 0) a.scale_t[blockIdx.x * a.scale_t_ld + blockIdx.y] = (uint8_t)ball;
        __syncthreads();
        // codes_t_ld is a multiple of 16: pieces of 16 rows, zeros behind the last row
        const int64_t rend = (a.rows + 15) / 16 * 16;
#pragma unroll
        for (int p = threadIdx.x; p < BLK * 8; p += 256) {
            const int col = p >> 3, piece = p & 7, x = (col >> 3) & 15;
            if (c0 + col < a.cols && r0 + 16 * piece < rend) {
                uint2 q[2];
                q[0] = *(const uint2 *)&tr[col * 32 + 2 * ((2 * piece) ^ x)];
                q[1] = *(const uint2 *)&tr[col * 32 + 2 * ((2 * piece + 1) ^ x)];
                __builtin_memcpy(a.codes_t + (c0 + col) * a.codes_t_ld + r0 + 16 * piece, q, 16);
            }
        }
    }
    if (a.sums) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float s = 0.f;
#pragma unroll
            for (int r = 0; r < 8; ++r) s += v[r][j];
            red[i][8 * l + j] = s;
        }
        __syncthreads();
        if (threadIdx.x < BLK && c0 + threadIdx.x < a.cols) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < 16; ++k) s += red[k][threadIdx.x];
            a.sums[(int64_t)blockIdx.y * a.cols + c0 + threadIdx.x] = s;
        }
    }
}

// Codes of any pitch and alignment to a pitch y_ld that is a multiple of 16, zeros behind the last
// column: up to two matrices in a launch.
struct RepackArgs {
    const uint8_t *x[2];
    uint8_t *y[2];
    int64_t rows[2], ld[2];
    int64_t cols, y_ld;
};
__global__ __launch_bounds__(256) void k_repack(RepackArgs a) {
    const int64_t np = a.y_ld / 16, first = a.rows[0] * np, total = first + a.rows[1] * np;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int which = i >= first;
        const int64_t p = which ? i - first : i, row = p / np, c = p % np * 16;
        const uint8_t *x = a.x[which] + row * a.ld[which] + c;
        uint8_t q[16];
        if (c + 16 <= a.cols) {
            __builtin_memcpy(q, x, 16);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) q[j] = c + j < a.cols ? x[j] : 0;
        }
        __builtin_memcpy(a.y[which] + row * a.y_ld + c, q, 16);
    }
}

// ------------------------------------------------------------ product
struct MatArgs {
    const uint8_t *a, *b;    // codes [M][K], [N][K]; pitches and K multiples of 16 for the tile kernels
    const uint8_t *sa, *sb;  // scale bytes
    const float *bias;       // [N], nullable
    void *out;
    float *part;             // [splits][M][N] where the contraction is split
    int64_t M, N, K, lda, ldb, lsa, lsb, ldo;
    int sha, shb;            // log2 of the rows that share a scale: 0 or 7
    int ksteps;              // blocks of 128 along K
    int kper;                // of them for each split
    int tm, tn;              // tiles
};

// LDS tiles of the tile kernels: rows of one block, 128 bytes; granule (16 bytes) g of row r
// stands at g ^ swz(r).  v_mfma_scale_f32_32x32x64_f8f6f4 takes half a block, a lane 32 bytes of
// one row (the order of k is free as long as both operands have the same): granules h and h + 2
// of the half, h = lane / 32.  With this swizzle the 16 lanes of each pass of a ds_read_b128 (rows
// 0-3, 12-15, 20-27, then the others) fall on 16 different 16-byte banks.
__device__ __forceinline__ int swz(int r) { return (r >> 1) & 7; }

// 16 bytes a lane from base + off + soff to LDS, 1 KB a wave in lane order; zeros from size on.
// As assembly, because the compiler would let every read of LDS wait for all such loads
// that are on their way; the kernel waits for them itself, by their number.
// to: LDS address.
__device__ __forceinline__ int lds_address(const void *p) {
    return __builtin_amdgcn_readfirstlane((int)(uintptr_t)(const __attribute__((address_space(3))) char *)p);
}
__device__ __forceinline__ void load_lds(const uint8_t *base, int size, int to, int off, int soff) {
    const uint64_t p = (uint64_t)base;
    // (the same in all lanes: scalar registers)
    const i32x4 r = {__builtin_amdgcn_readfirstlane((int)(uint32_t)p),
                     __builtin_amdgcn_readfirstlane((int)((uint32_t)(p >> 32) & 0xffffu)),
                     __builtin_amdgcn_readfirstlane(size), 0x00027000};
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(off), "s"(r),
                 "s"(soff)
                 : "memory");
}

// c += 2^(sa + sb) a b^T for lanes' fragments fb (rows of b: the tile's rows) and fa (rows of
// a: its columns): 128 codes of a 16x16 tile, or 64 of a 32x32 one.  S: the scale's byte.
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
struct Wide { bf16x8 v[4]; };  // 32 codes as bf16, their scale applied
__device__ __forceinline__ Wide widen(const i32x8 &f, uint32_t s) {
    const float scale = scale_of((int)(s & 255u));
    Wide w;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)f[j], scale, false);
        const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)f[j], scale, true);
        w.v[j / 2][4 * (j & 1)] = lo[0];
        w.v[j / 2][4 * (j & 1) + 1] = lo[1];
        w.v[j / 2][4 * (j & 1) + 2] = hi[0];
        w.v[j / 2][4 * (j & 1) + 3] = hi[1];
    }
    return w;
}
__device__ __forceinline__ f32x4 block_product(const Wide &b, const Wide &a, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.v[j], a.v[j], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x16 block_product(const Wide &b, const Wide &a, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b.v[j], a.v[j], c, 0, 0, 0);
    return c;
}
struct Codes { i32x8 v; uint32_t s; };
template <int S = 0> __device__ __forceinline__ f32x16 block_product(const Codes &b, const Codes &a, f32x16 c) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b.v, a.v, c, 0, 0, S, (int)b.s, S, (int)a.s);
}
__device__ __forceinline__ f32x4 block_product(const Codes &b, const Codes &a, f32x4 c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.v, a.v, c, 0, 0, 0, (int)b.s, 0, (int)a.s);
}
// a fragment as the product of an output type takes it
template <typename TO> struct Operand {
    typedef Codes type;
    static __device__ __forceinline__ Codes of(const i32x8 &f, uint32_t s, int byte = 0) { return Codes{f, s}; }
};
template <> struct Operand<float> {
    typedef Wide type;
    static __device__ __forceinline__ Wide of(const i32x8 &f, uint32_t s, int byte = 0) { return widen(f, s >> (8 * byte)); }
};
// a step of a 32x32 tile with byte S of the scale words
template <int S> __device__ __forceinline__ f32x16 step_product(const Codes &b, const Codes &a, f32x16 c) {
    return block_product<S>(b, a, c);
}
template <int S> __device__ __forceinline__ f32x16 step_product(const Wide &b, const Wide &a, f32x16 c) {
    return block_product(b, a, c);
}

// four scale bytes kb .. kb+3 of a row, those from n on 0 (their codes are zeros)
__device__ __forceinline__ uint32_t scales4(const uint8_t *row, int kb, int n) {
    uint32_t s = 0;
    if (kb + 4 <= n) {
        __builtin_memcpy(&s, row + kb, 4);
    } else {
        for (int j = 0; j < 3; ++j)
            if (kb + j < n) s |= (uint32_t)row[kb + j] << (8 * j);
    }
    return s;
}

template <typename TO> __device__ __forceinline__ void st_out4(TO *p, const f32x4 &v, int64_t left) {
    const float t[4] = {v[0], v[1], v[2], v[3]};
    if (left >= 4) {
        st_vec<TO, 4>(p, t);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < left) p[j] = (TO)t[j];
    }
}

// Workgroups go round the 8 XCDs in turn, each with an L2 of its own: an XCD takes a
// contiguous run of tiles, in bands of 8 tile rows, so that the tiles it works on at a
// time share their rows of a and of b.
__device__ __forceinline__ void tile_of(int id, int tm, int tn, int &im, int &in) {
    const int n = tm * tn, per = n / 8, rest = n % 8, xcd = id % 8, k = id / 8;
    const int t = xcd * per + (xcd < rest ? xcd : rest) + k;
    const int band = 8 * tn, b = t / band, h = tm - 8 * b < 8 ? tm - 8 * b : 8;
    im = 8 * b + (t - b * band) % h;
    in = (t - b * band) / h;
}

// A workgroup of WM x WN waves computes BM x BN outputs, a wave BM/WM x BN/WN of them in
// 32x32 tiles.  What keeps the matrix cores fed:
//   - the blocks of the next step travel from memory to LDS without registers while a step is
//     multiplied (two stages); whole 128-byte lines, since the L1 fetches no less;
//   - a wave reads the fragments of the next half block while it multiplies those of this
//     one, so that a step's one barrier waits for nothing that was just asked for;
//   - waves of 128 x 128 outputs (4 of them, one a SIMD): every fragment is used four times.  A
//     CU reads 128 bytes of LDS a cycle: waves of 128 x 64 would read as long as they multiply.
// A step is one run of instructions without a branch, in which the compiler keeps to rows of tiles:
// loads and reads are issued between matrix instructions, which hide them.  Scales are fetched 16
// steps at a time (a row's 16 bytes; every fetch costs a line of the L1) and read from LDS step by step.
// The outputs leave through LDS in whole rows.
// Bound by the matrix cores where the contraction is long: 8192^3 400-428 us, 2.6-2.75 PFLOP/s (0.87-0.93 of
// the library's 8-bit product with one scale a tensor); 4096^3 57 us, 2.4.  Short contractions are bound by the
// tile's beginning and end: 50240 x 1536, K = 384, 72 us, 0.82, of which the outputs' bytes are 30.  fp32 outputs 4096^3 118 us, 1.17 (the
// library's bf16 product 1.34-1.46).
template <int BM, int BN, int WM, int WN, typename TO>
__global__ __launch_bounds__(64 * WM * WN, 1) void k_block_matmul(MatArgs a) {
    constexpr int WAVES = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, STAGE = (BM + BN) * BLK;
    constexpr int LA = BM / 8 / WAVES, LB = BN / 8 / WAVES;  // loads of 1 KB, 8 rows, a wave and step
    constexpr int SR = (BM + BN) / (64 * WAVES);             // rows whose scales a thread fetches
    constexpr bool SPLITS = BM == 128;                       // fp32 parts fit the stages
    static_assert(BM % 64 == 0 && SR >= 1, "a wave fetches scales of a or of b");
    static_assert(WAVES % 2 == 0, "bit 3 of a load's first row is the wave's lowest");
    static_assert(BM * BN * (SPLITS ? 4 : (int)sizeof(TO)) <= 2 * STAGE, "the outputs fit the stages");
    constexpr int SG = 16;                                   // steps of a fetch of scales
    __shared__ __align__(16) char buf[2 * STAGE];
    __shared__ uint8_t sc[2][SG][BM + BN];
    __shared__ __align__(16) float sbias[BN];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN, h = lane >> 5, i32 = lane & 31;
    int im, in;
    tile_of(blockIdx.x, a.tm, a.tn, im, in);
    const int64_t m0 = (int64_t)im * BM, n0 = (int64_t)in * BN;
    const int kb0 = blockIdx.y * a.kper, kb1 = kb0 + a.kper < a.ksteps ? kb0 + a.kper : a.ksteps;
    // bytes of the contraction that this workgroup takes, from kb0 * BLK on
    const int klen = (int)((int64_t)kb1 * BLK < a.K ? (int64_t)(kb1 - kb0) * BLK : a.K - (int64_t)kb0 * BLK);
    const int steps = kb1 - kb0;
    const int arows = a.M - m0 < BM ? (int)(a.M - m0) : BM, brows = a.N - n0 < BN ? (int)(a.N - n0) : BN;
    const uint8_t *abase = a.a + m0 * a.lda + (int64_t)kb0 * BLK, *bbase = a.b + n0 * a.ldb + (int64_t)kb0 * BLK;
    const int asize = (int)((arows - 1) * a.lda) + klen, bsize = (int)((brows - 1) * a.ldb) + klen;
    // this lane's granule in each of its loads; rows behind the matrix: out of any range, read as zeros
    constexpr int OUT = 0x7fffffff;
    int off[LA + LB];
    const int g16 = 16 * ((lane & 7) ^ swz((wave & 1) * 8 + (lane >> 3)));
#pragma unroll
    for (int i = 0; i < LA + LB; ++i) {
        const bool isa = i < LA;
        const int r = ((isa ? i : i - LA) * WAVES + wave) * 8 + (lane >> 3);
        off[i] = r < (isa ? arows : brows) ? (int)(r * (isa ? a.lda : a.ldb)) + g16 : OUT;
    }
    const int lds = lds_address(buf) + wave * 1024;
    auto load = [&](int s, int i) {  // load i of step s; behind the last step nothing is read (a size of 0)
        const bool live = s < steps;
        const int to = lds + (s & 1) * STAGE + (i < LA ? i * WAVES * 1024 : BM * BLK + (i - LA) * WAVES * 1024);
        load_lds(i < LA ? abase : bbase, live ? (i < LA ? asize : bsize) : 0, to, off[i], live ? s * BLK : 0);
    };
    auto cut = [&] {  // before the loads of the last step: what lies behind the row's last code is not read
        if ((steps - 1) * BLK + g16 >= klen) {
#pragma unroll
            for (int i = 0; i < LA + LB; ++i) off[i] = OUT;
        }
    };
    const uint8_t *sp[SR];
#pragma unroll
    for (int i = 0; i < SR; ++i) {
        const int r = i * 64 * WAVES + (int)threadIdx.x, rb = r - BM;
        if (r < BM) sp[i] = a.sa + ((m0 + (r < arows ? r : arows - 1)) >> a.sha) * a.lsa;
        else sp[i] = a.sb + ((n0 + (rb < brows ? rb : brows - 1)) >> a.shb) * a.lsb;
    }
    i32x4 word[SR];
    auto fetch_scales = [&](int s) {  // of steps s .. s+15; those behind the last are not used
#pragma unroll
        for (int i = 0; i < SR; ++i) {
            if (s + SG <= steps) {
                __builtin_memcpy(&word[i], sp[i] + kb0 + s, SG);
            } else {  // bytes, none behind the row's last: all on their way at once
                uint8_t b[SG];
#pragma unroll
                for (int j = 0; j < SG; ++j) b[j] = sp[i][kb0 + (s + j < steps ? s + j : steps - 1)];
                __builtin_memcpy(&word[i], b, SG);
            }
        }
    };
    auto put_scales = [&](int s) {
#pragma unroll
        for (int i = 0; i < SR; ++i)
#pragma unroll
            for (int j = 0; j < SG; ++j)
                sc[(s / SG) & 1][j][i * 64 * WAVES + threadIdx.x] = (uint8_t)(word[i][j >> 2] >> (8 * (j & 3)));
    };
    uint32_t sa[TM], sb[TN], na[TM], nb[TN];  // of this step and the next
    auto read_scales = [&](int s) {
        const uint8_t *p = &sc[(s / SG) & 1][s % SG][i32];
#pragma unroll
        for (int i = 0; i < TM; ++i) na[i] = p[(wm * TM + i) * 32];
#pragma unroll
        for (int j = 0; j < TN; ++j) nb[j] = p[BM + (wn * TN + j) * 32];
    };
    // fragments of half u of a stage: rows of 32, granules 4u + h and 4u + h + 2
    const int fo = i32 * BLK + 16 * (h ^ swz(i32));
    const int fa = wm * TM * 32 * BLK + fo, fb = (BM + wn * TN * 32) * BLK + fo;
    auto fragment = [&](const char *tile, int at) {
        const i32x4 lo = *(const i32x4 *)(tile + at), hi = *(const i32x4 *)(tile + (at ^ 32));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    i32x8 ca[2][TM], cb[2][TN];
    auto read = [&](const char *stage, auto U, int k) {  // fragment k of a half: those of b, then of a
        constexpr int u = U;
        if (k < TN) cb[u][k] = fragment(stage + k * 32 * BLK, fb ^ (64 * u));
        else ca[u][k - TN] = fragment(stage + (k - TN) * 32 * BLK, fa ^ (64 * u));
    };
    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    // One half: a row of tiles at a time, and between them what `with` issues, which the
    // matrix instructions of the row (TN of 64 cycles) hide.  The compiler keeps to the rows.
    auto multiply = [&](auto U, auto with) {
        constexpr int u = U;
        typename Operand<TO>::type wb[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            with(i);
            if (i == 0) {
#pragma unroll
                for (int j = 0; j < TN; ++j) wb[j] = Operand<TO>::of(cb[u][j], sb[j]);
            }
            const typename Operand<TO>::type wa = Operand<TO>::of(ca[u][i], sa[i]);
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = block_product(wb[j], wa, acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr std::integral_constant<int, 0> first{};
    constexpr std::integral_constant<int, 1> second{};
    constexpr int HALF = TM / 2;                             // reads go with the first rows: done by the barrier
    constexpr int READS = (TM + TN + HALF - 1) / HALF, LOADS = (LA + LB + TM - 1) / TM;  // with each row
    // (32 loads a lane where the outputs leave took a fifth of a short contraction's time)
    float bias = 0.f;
    if (a.bias && !a.part) bias = a.bias[n0 + (int)threadIdx.x < a.N ? n0 + threadIdx.x : a.N - 1];
    if (steps == 1) cut();
#pragma unroll
    for (int i = 0; i < LA + LB; ++i) load(0, i);
    if (steps == 2) cut();
#pragma unroll
    for (int i = 0; i < LA + LB; ++i) load(1, i);
    fetch_scales(0);
    if ((int)threadIdx.x < BN) sbias[threadIdx.x] = bias;
    put_scales(0);  // (waits for the words, and so for the loads before them)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int k = 0; k < TM + TN; ++k) read(buf, first, k);
    read_scales(0);
    for (int s = 0; s < steps;) {
        if (s % SG == 0) {
            if (s == 0 && SG < steps) fetch_scales(SG);
            if (s + SG < steps) put_scales(s + SG);
            if (s + 2 * SG < steps) fetch_scales(s + 2 * SG);
        }
        if (s == steps - 3) cut();
        int end = s - s % SG + SG < steps ? s - s % SG + SG : steps;
        if (s < steps - 3 && end > steps - 3) end = steps - 3;
#pragma clang loop unroll(disable)
        for (; s < end; ++s) {
            const char *cur = buf + (s & 1) * STAGE, *nxt = buf + (~s & 1) * STAGE;
#pragma unroll
            for (int i = 0; i < TM; ++i) sa[i] = na[i];
#pragma unroll
            for (int j = 0; j < TN; ++j) sb[j] = nb[j];
            multiply(first, [&](int i) {
#pragma unroll
                for (int k = i * READS; k < (i + 1) * READS && k < TM + TN; ++k) read(cur, second, k);
            });
            // the next step is in LDS, and every wave has read this one
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            multiply(second, [&](int i) {
#pragma unroll
                for (int k = i * READS; k < (i + 1) * READS && k < TM + TN; ++k) read(nxt, first, k);
#pragma unroll
                for (int k = i * LOADS; k < (i + 1) * LOADS && k < LA + LB; ++k) load(s + 2, k);
                if (i == HALF) read_scales(s + 1);
            });
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the stages are read, and no load is on its way
    // Outputs through LDS.  A lane holds column i32 of each tile (a row of a) and rows 8 e + 4 h .. + 3
    // (rows of b).  A wave's rows have their granules swizzled by the row: 16 lanes' pieces of 16
    // rows in 16 banks.  EO: the stored type, of out or of a part.
    auto store = [&](auto *out, int64_t ldo, auto put) {
        typedef std::remove_pointer_t<decltype(out)> EO;
        constexpr int ROW = BN / WN * (int)sizeof(EO), G = ROW / 16, RPI = 64 / G, PIECE = 16 / (int)sizeof(EO);
        char *mine = buf + wave * (TM * 32 * ROW);
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = j * 32 + 8 * e + 4 * h;
                const f32x4 bias = *(const f32x4 *)(sbias + wn * TN * 32 + c);
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const float t[4] = {acc[i][j][4 * e] + bias[0], acc[i][j][4 * e + 1] + bias[1],
                                        acc[i][j][4 * e + 2] + bias[2], acc[i][j][4 * e + 3] + bias[3]};
                    const int byte = c * (int)sizeof(EO), r = i * 32 + i32;
                    char *p = mine + r * ROW + 16 * ((byte / 16) ^ (r & (G - 1))) + byte % 16;
                    st_vec<EO, 4>((EO *)__builtin_assume_aligned(p, 4 * sizeof(EO)), t);
                }
            }
        const int g = lane % G;
        const int64_t n = n0 + wn * TN * 32 + g * PIECE;
#pragma unroll 4
        for (int i = 0; i < TM * 32 / RPI; ++i) {
            const int r = i * RPI + lane / G;
            const int64_t m = m0 + wm * TM * 32 + r;
            const i32x4 v = *(const i32x4 *)(mine + r * ROW + 16 * (g ^ (r & (G - 1))));
            if (m >= a.M) continue;
            EO *p = out + m * ldo + n;
            if (n + PIECE <= a.N) {
                put(p, v);
            } else {
                EO t[PIECE];
                __builtin_memcpy(t, &v, 16);
#pragma unroll
                for (int k = 0; k < PIECE; ++k)
                    if (n + k < a.N) p[k] = t[k];
            }
        }
    };
    if constexpr (SPLITS) {
        if (a.part)
            return store(a.part + (int64_t)blockIdx.y * a.M * a.N, a.N, [](float *p, i32x4 v) { __builtin_memcpy(p, &v, 16); });
    }
    store((TO *)a.out, a.ldo, [](TO *p, i32x4 v) { st_stream(p, v); });
}

// The parts of a split contraction, added in order, with the bias.  Bound by memory (1536 x 384 of 14 parts:
// 7.5 us with the launch).
template <typename TO> __global__ __launch_bounds__(256) void k_split_sum(MatArgs a, int splits) {
    const int64_t total = a.M * a.N, stride = (int64_t)gridDim.x * 256 * 4;
    for (int64_t p = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; p < total; p += stride) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        for (int z = 0; z < splits; ++z) {
            float t[4];
            ld_row<float, 4>(a.part + z * total, p, total, t);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += t[e];
        }
        const int64_t m = p / a.N, n = p % a.N;
        if (n + 4 <= a.N) {
            if (a.bias)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += a.bias[n + e];
            st_vec<TO, 4>((TO *)a.out + m * a.ldo + n, s);
        } else {
            for (int e = 0; e < 4 && p + e < total; ++e) {
                const int64_t me = (p + e) / a.N, ne = (p + e) % a.N;
                ((TO *)a.out)[me * a.ldo + ne] = (TO)(s[e] + (a.bias ? a.bias[ne] : 0.f));
            }
        }
    }
}

// ------------------------------------------------------------ few rows
// Up to 32 rows of a (single tokens): bound by the bytes of b, which no two workgroups
// share.  A workgroup owns 16 rows of b; its 8 waves split the contraction (and, where
// that leaves the chip empty, so does the grid), read b from memory straight into the
// matrix cores' operands (a lane 32 consecutive bytes of a row, 128 bytes a row and
// instruction), and add their tiles through LDS in the waves' order.
// QUANT (up to 16 rows): a is bf16 or fp32 and is quantised on the way (its blocks' 128 values
// are in 4 lanes), which saves the quantiser's launch; every workgroup repeats it for its share.
// Weights from memory, us: one row 4096 x 4096 7.7, 8192 x 8192 16 (codes alone; 4.2 TB/s); 16 rows 4096 x
// 4096 10.4, of which 2.5 is quantising; 32 rows 13.4.  2304 x 768, one row: 3.3, a launch's latency.
struct SkinnyArgs {
    MatArgs m;
    const void *x;
    int64_t ldx;
};

template <int MT, typename TX, bool QUANT, typename TO>
__global__ __launch_bounds__(512) void k_block_matmul_few(SkinnyArgs s) {
    const MatArgs &a = s.m;
    constexpr int WAVES = 8;
    __shared__ f32x4 red[WAVES - 1][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int q = lane >> 4, i16 = lane & 15;
    const int64_t n = (int64_t)blockIdx.x * 16 + i16, nc = n < a.N ? n : a.N - 1;
    const uint8_t *brow = a.b + nc * a.ldb, *sbrow = a.sb + (nc >> a.shb) * a.lsb;
    const int kb0 = blockIdx.y * a.kper, kb1 = kb0 + a.kper < a.ksteps ? kb0 + a.kper : a.ksteps;
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    // 32 bytes k .. k+31 of a row of codes, zeros from K on
    auto codes32 = [&](const uint8_t *row, int64_t k) {
        i32x8 f;
        if (no_lane(k + 32 > a.K)) {
            __builtin_memcpy(&f, row + k, 32);
        } else {
            const int left = left_in_row<32>(k, a.K);
            const uint8_t *p = row + (left ? k : 0);
            uint8_t t[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) t[j] = p[j < left ? j : 0];
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                uint32_t v = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) v |= (4 * w + j < left ? (uint32_t)t[4 * w + j] : 0u) << (8 * j);
                f[w] = (int)v;
            }
        }
        return f;
    };
    // U blocks of b are on their way at once, and of 16 rows of a.  (Whether there is a block is the
    // wave's own: the branches are uniform.)
    constexpr int U = 4;
    for (int kb = kb0 + wave; kb < kb1; kb += WAVES * U) {
        i32x8 fb[U];
        uint32_t sb[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kc = kb + u * WAVES;
            if (kc >= kb1) break;
            fb[u] = codes32(brow, (int64_t)kc * BLK + 32 * q);
            sb[u] = sbrow[kc];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int64_t m = 16 * i + i16, mc = m < a.M ? m : a.M - 1;
            std::conditional_t<QUANT, Eight<TX>, int> x[U][4];
            i32x8 fa[U];
            uint32_t sa[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int kc = kb + u * WAVES;
                if (kc >= kb1) break;
                const int64_t k = (int64_t)kc * BLK + 32 * q;
                if constexpr (QUANT) {
                    const TX *row = (const TX *)s.x + mc * s.ldx;
#pragma unroll
                    for (int p = 0; p < 4; ++p) x[u][p].load(row, k + 8 * p, a.K);
                } else {
                    fa[u] = codes32(a.a + mc * a.lda, k);
                    sa[u] = a.sa[(mc >> a.sha) * a.lsa + kc];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (kb + u * WAVES >= kb1) break;
                if constexpr (QUANT) {
                    float amax = 0.f;
#pragma unroll
                    for (int p = 0; p < 4; ++p) amax = fmaxf(amax, x[u][p].amax());
                    amax = fmaxf(amax, __shfl_xor(amax, 16, 64));
                    amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
                    sa[u] = (uint32_t)scale_byte(amax);
                    const float scale = scale_of((int)sa[u]);
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        uint32_t c[2];
                        x[u][p].codes(scale, c);
                        fa[u][2 * p] = (int)c[0];
                        fa[u][2 * p + 1] = (int)c[1];
                    }
                }
                acc[i] = block_product(Operand<TO>::of(fb[u], sb[u]), Operand<TO>::of(fa[u], sa[u]), acc[i]);
            }
        }
    }
    if (wave > 0) {
#pragma unroll
        for (int i = 0; i < MT; ++i) red[wave - 1][i][lane] = acc[i];
    }
    __syncthreads();
    if (wave > 0) return;
    const int64_t n4 = (int64_t)blockIdx.x * 16 + 4 * q;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int w = 0; w < WAVES - 1; ++w) acc[i] += red[w][i][lane];
        const int64_t m = 16 * i + i16;
        if (m >= a.M || n4 >= a.N) continue;
        if (a.part) {
            st_out4<float>(a.part + ((int64_t)blockIdx.y * a.M + m) * a.N + n4, acc[i], a.N - n4);
        } else {
            if (a.bias)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][e] += n4 + e < a.N ? a.bias[n4 + e] : 0.f;
            st_out4<TO>((TO *)a.out + m * a.ldo + n4, acc[i], a.N - n4);
        }
    }
}

}  // namespace race
