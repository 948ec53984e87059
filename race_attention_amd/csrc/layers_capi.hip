// layers_capi.hip -- the extern "C" boundary of the operators around RACE attention:
// root-mean-square norm, matrices in 8-bit blocks and their product, AdamW
// (include/race_attention.h).  As in race_capi.hip every argument is checked on the host
// before a launch, nothing is allocated and calls run on the caller's stream.
#include "../../include/race_attention.h"
#include "adamw.hip"
#include "block_fp8.hip"
#include "race_error.h"
#include "rms_norm.hip"

#include <cmath>

namespace race {
namespace {

typedef long long ll;

bool dtype_ok(int t) { return t == RACE_DTYPE_F32 || t == RACE_DTYPE_BF16; }
int esize(int t) { return t == RACE_DTYPE_BF16 ? 2 : 4; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// a pointer of elements of es bytes
int check_ptr(const char *name, const void *p, int es) {
    if (!p) return fail(RACE_E_INVALID, "%s is NULL", name);
    if ((uintptr_t)p % es) return fail(RACE_E_INVALID, "%s is not %d-byte aligned", name, es);
    return RACE_OK;
}
// rows of n elements es bytes each, stride elements apart; one that is written has rows that do not overlap
int check_rows(const char *name, const void *p, int es, int64_t rows, int64_t n, int64_t stride, bool written) {
    if (int rc = check_ptr(name, p, es)) return rc;
    if (stride < 0 || (written && rows > 1 && stride < n))
        return fail(RACE_E_INVALID, "%s row stride %lld of %lld columns", name, (ll)stride, (ll)n);
    return RACE_OK;
}

// ------------------------------------------------------------ norm
int check_norm(const race_norm_desc *d) {
    if (!d) return fail(RACE_E_INVALID, "descriptor is NULL");
    if (!dtype_ok(d->dtype) || !dtype_ok(d->r_dtype))
        return fail(RACE_E_INVALID, "dtype %d or r_dtype %d is not RACE_DTYPE_F32 or RACE_DTYPE_BF16", d->dtype, d->r_dtype);
    if (d->dtype == RACE_DTYPE_F32 && d->r_dtype == RACE_DTYPE_BF16)
        return fail(RACE_E_UNSUPPORTED, "an fp32 x with a bf16 residual: the sum would lose x's bits");
    if (d->rows < 1 || d->D < 1) return fail(RACE_E_INVALID, "rows and D must be >= 1 (got %lld, %lld)", (ll)d->rows, (ll)d->D);
    if (d->D > ((int64_t)1 << 30)) return fail(RACE_E_UNSUPPORTED, "D=%lld columns unsupported (D <= 2^30)", (ll)d->D);
    if (!(d->eps >= 0.f) || d->eps > 1e30f) return fail(RACE_E_INVALID, "eps must be finite and >= 0");
    return RACE_OK;
}

// Workgroups of a launch: rows beyond them are walked.  2^20 of 256 threads keep the
// launch's work-items within 32 bits.
unsigned norm_grid(int64_t rows, int rpb) {
    const int64_t n = ceil_div(rows, rpb);
    return (unsigned)(n < (1 << 20) ? n : 1 << 20);
}
// of the backward, each with a row of dw_part: as many as keep the memory busy, and no more, because
// their parts are written and added.  us at 512, 768 and 1024: 65536 x 768 bf16 100, 101, 111; 8192 x
// 4096 67, 77, 73; 4001 x 1001 fp32 17, 20, 23; 50240 x 384 fp32 104, 87, 82 (short rows: little of one is on
// its way at a time).
int64_t norm_bwd_grid(int64_t rows, int64_t D) {
    const int64_t n = ceil_div(rows, D <= 1024 ? 4 : 1), most = D <= 512 ? 1024 : 512;
    return n < most ? n : most;
}

// f<V, NV, L>() for a row length: a wave up to 1024 columns, a workgroup up to HELD.  To codes that is 4096:
// more columns a thread take the registers of the waves that would hide each other's loads (us, 16384 x 5120
// held and read twice: 188 and 160; 16384 x 8192 239 and 232; 8192 x 16384 509 and 243).
template <int HELD, typename F> void norm_config(int64_t D, F &&f) {
    const int n = (int)ceil_div(D, 256);
    if (D <= 1024) {
        if (n == 1) f(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 64>{});
        else if (n == 2) f(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{}, std::integral_constant<int, 64>{});
        else if (n == 3) f(std::integral_constant<int, 4>{}, std::integral_constant<int, 3>{}, std::integral_constant<int, 64>{});
        else f(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{}, std::integral_constant<int, 64>{});
    } else {
        if (D <= 2048) f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 256>{});
        else if (D <= 4096) f(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{}, std::integral_constant<int, 256>{});
        else {
            if constexpr (HELD > 4096) {
                if (D <= 8192) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{}, std::integral_constant<int, 256>{});
                if (D <= HELD) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 8>{}, std::integral_constant<int, 256>{});
            }
            f(std::integral_constant<int, 8>{}, std::integral_constant<int, 0>{}, std::integral_constant<int, 256>{});
        }
    }
}
// f<TX, TR>()
template <typename F> void norm_types(int x, int r, F &&f) {
    if (x == RACE_DTYPE_F32) f(float{}, float{});
    else if (r == RACE_DTYPE_F32) f(bf16{}, float{});
    else f(bf16{}, bf16{});
}

int norm_forward(const race_norm_desc *d, const void *x, const void *residual, const float *w, void *y, bool codes,
                 uint8_t *scale, int64_t scale_stride, void *h, float *rstd, void *stream, const char *what) {
    if (int rc = check_norm(d)) return rc;
    const int ex = esize(d->dtype), er = esize(d->r_dtype);
    int rc;
    if ((rc = check_rows("x", x, ex, d->rows, d->D, d->x_stride, false)) || (rc = check_ptr("w", w, 4)) ||
        (rc = check_rows(codes ? "codes" : "y", y, codes ? 1 : ex, d->rows, d->D, d->y_stride, true)))
        return rc;
    if (!residual != !h) return fail(RACE_E_INVALID, "residual and h are given together or not at all");
    if (residual && ((rc = check_rows("residual", residual, er, d->rows, d->D, d->r_stride, false)) ||
                     (rc = check_rows("h", h, er, d->rows, d->D, d->h_stride, true))))
        return rc;
    if (codes && (rc = check_rows("scale", scale, 1, d->rows, ceil_div(d->D, BLK), scale_stride, true))) return rc;
    if (rstd && (rc = check_ptr("rstd", rstd, 4))) return rc;
    NormArgs a{};
    a.x = x;
    a.r = residual;
    a.w = w;
    a.y = y;
    a.h = h;
    a.scale = scale;
    a.rstd = rstd;
    a.rows = d->rows;
    a.D = d->D;
    a.xs = d->x_stride;
    a.rs = d->r_stride;
    a.ys = d->y_stride;
    a.hs = d->h_stride;
    a.ss = scale_stride;
    a.eps = d->eps;
    hipStream_t s = (hipStream_t)stream;
    norm_types(d->dtype, residual ? d->r_dtype : d->dtype, [&](auto tx, auto tr) {
        auto launch = [&](auto V, auto NV, auto L, auto to_codes) {
            const unsigned grid = norm_grid(d->rows, NORM_THREADS / L);
            k_rms_norm<decltype(tx), decltype(tr), V, NV, L, to_codes><<<grid, NORM_THREADS, 0, s>>>(a);
        };
        if (codes) norm_config<4096>(d->D, [&](auto V, auto NV, auto L) { launch(V, NV, L, std::true_type{}); });
        else norm_config<16384>(d->D, [&](auto V, auto NV, auto L) { launch(V, NV, L, std::false_type{}); });
    });
    return launched(what);
}

// ------------------------------------------------------------ 8-bit blocks
int check_blocks(const char *name, const race_blocks *b) {
    if (!b) return fail(RACE_E_INVALID, "%s is NULL", name);
    if (b->rows < 1 || b->cols < 1)
        return fail(RACE_E_INVALID, "%s: rows and cols must be >= 1 (got %lld, %lld)", name, (ll)b->rows, (ll)b->cols);
    if (b->rows > ((int64_t)1 << 31) - 256 || b->cols > ((int64_t)1 << 31) - 256)
        return fail(RACE_E_UNSUPPORTED, "%s: %lld x %lld exceeds 2^31 rows or columns", name, (ll)b->rows, (ll)b->cols);
    if (b->block_rows != 1 && b->block_rows != BLK)
        return fail(RACE_E_INVALID, "%s: a scale is shared by 1 or 128 rows (got %d)", name, b->block_rows);
    if (!b->codes || !b->scale) return fail(RACE_E_INVALID, "%s: codes or scale is NULL", name);
    if (b->ld < b->cols || b->scale_ld < ceil_div(b->cols, BLK))
        return fail(RACE_E_INVALID, "%s: row pitch %lld (scales %lld) of %lld columns", name, (ll)b->ld, (ll)b->scale_ld,
                    (ll)b->cols);
    return RACE_OK;
}
// blocks that a quantiser writes: pitch of whole 16-byte pieces
int check_out_blocks(const char *name, const race_blocks *b) {
    if (int rc = check_blocks(name, b)) return rc;
    if (b->ld % 16 || b->ld < round_up(b->cols, 16) || (uintptr_t)b->codes % 16)
        return fail(RACE_E_INVALID, "%s: codes and their pitch must be whole 16-byte pieces", name);
    return RACE_OK;
}

struct MatPlan {
    int M, N;            // rows of a, of b
    int64_t K;           // contraction, as the kernels see it
    int ksteps, few;     // blocks along K; few: the kernel for few rows
    int bm, bn, tm, tn, splits, kper;
    size_t pack_a, pack_b, parts;  // workspace: repacked operands, parts of a split contraction
};

// Rows of a up to which k_block_matmul_few multiplies: beyond them tiles of 128 are as fast or faster (64
// rows in tiles and as few: 4096 x 4096 19 and 17 us, 8192 x 8192 26 and 55).  And the rows that
// race_block_linear takes, of 16-bit or 32-bit numbers.
constexpr int kFewRows = 32, kLinearRows = 16;
constexpr int kCUs = 256;

bool direct(const race_blocks *b) { return b->ld % 16 == 0 && b->cols % 16 == 0 && (uintptr_t)b->codes % 16 == 0; }
// Whether the few rows' kernel quantises by itself, or a launch before it does: every workgroup (16 rows
// of b) repeats the former's work, while the latter costs its launch.  us, the former and the latter, 1 and 16
// rows, weights from memory, launches of a graph: 768 x 768 3.0 / 4.3, 3.6 / 5.0; 4096 x 4096 7.7 / 8.3,
// 10.4 / 10.5; 1024 x 8192 9.8 / 9.6, 16.2 / 13.8; 8192 x 4096 14.3 / 12.9, 19.3 / 17.0; 32768 x 1024
// 19.5 / 17.7, 24.2 / 21.8.
bool quantise_first(const race_blocks *b) { return b->cols > 4096 || b->rows * b->cols > (1 << 24); }
size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

int mat_plan(const race_blocks *a, const race_blocks *b, int out_dtype, MatPlan &p) {
    int rc;
    if ((rc = check_blocks("a", a)) || (rc = check_blocks("b", b))) return rc;
    if (!dtype_ok(out_dtype)) return fail(RACE_E_INVALID, "out_dtype %d is not RACE_DTYPE_F32 or RACE_DTYPE_BF16", out_dtype);
    if (a->cols != b->cols) return fail(RACE_E_INVALID, "a has %lld columns, b %lld", (ll)a->cols, (ll)b->cols);
    p = MatPlan{};
    p.M = (int)a->rows;
    p.N = (int)b->rows;
    p.K = a->cols;
    p.ksteps = (int)ceil_div(p.K, BLK);
    p.few = p.M <= kFewRows;
    if (p.few) {
        p.tn = (int)ceil_div(p.N, 16);
        // Workgroups of 8 waves, one to 16 rows of b.  The sum of a split costs a launch, 4 us: it pays
        // where few workgroups would walk many blocks each.
        const int64_t want = ceil_div(kCUs, p.tn), most = ceil_div(p.ksteps, 8 * 8);
        p.splits = (int)(want < most ? want : most);
        if ((int64_t)p.tn * 512 * (p.splits < 1 ? 1 : p.splits) >= (int64_t)1 << 32)
            return fail(RACE_E_UNSUPPORTED, "%d rows of b exceed one launch's 2^32 work-items", p.N);
    } else {
        p.K = round_up(p.K, 16);
        if (!direct(a)) p.pack_a = align256((size_t)(a->rows * p.K));
        if (!direct(b)) p.pack_b = align256((size_t)(b->rows * p.K));
        const int64_t lda = p.pack_a ? p.K : a->ld, ldb = p.pack_b ? p.K : b->ld;
        if (lda >= (1 << 22) || ldb >= (1 << 22))
            return fail(RACE_E_UNSUPPORTED, "row pitch of 2^22 bytes or more (a %lld, b %lld)", (ll)lda, (ll)ldb);
        // Tiles of 256 x 256 (one workgroup a CU) feed the matrix cores better, 1.6 us a step
        // against 2 x 1.0 us of the four times smaller work of 128 x 128 (two a CU); but no other workgroup
        // works while one begins and ends, 10 us against 4.  128 x 128 may also split the contraction;
        // its parts are written and read once (4 TB/s) and take a launch.  The least estimate is taken.
        // us, 256 and 128: 8192^3 398 and 495; 4096^3 57 and 66; 4096 x 4096, K = 1024, 23.4 and 25.8; 50240 x 1536,
        // K = 384, 75 and 72; 50240 x 384, K = 1536, 53 and 45; 8192 x 2304, K = 768, 35 and 28; 2048 x 2048, K =
        // 8192, split, 79 and 46.  (fp32 outputs: the bf16 operands take 128 x 128's registers.)
        const int64_t big = ceil_div(p.M, 256) * ceil_div(p.N, 256), small = ceil_div(p.M, 128) * ceil_div(p.N, 128);
        double best = out_dtype == RACE_DTYPE_F32 ? 1e30 : (double)ceil_div(big, kCUs) * (1.6 * p.ksteps + 10);
        p.bm = 256;
        for (int s = 1; s == 1 || (s <= 64 && 2 * s <= p.ksteps && (s - 1) * small < 2 * kCUs); ++s) {
            const int64_t wgs = small * s;
            // (bf16 products of an fp32 output: 1.75 and 1.5)
            const double step = out_dtype == RACE_DTYPE_F32 ? (wgs <= kCUs ? 1.5 : 1.75) : wgs <= kCUs ? 0.65 : 1.0;
            const double t = (double)ceil_div(wgs, 2 * kCUs) * (step * ceil_div(p.ksteps, s) + 4) +
                             (s > 1 ? 4 + 2e-6 * s * p.M * p.N : 0.0);
            if (t < best) {
                best = t;
                p.bm = 128;
                p.splits = s;
            }
        }
        p.bn = p.bm;
        p.tm = (int)ceil_div(p.M, p.bm);
        p.tn = (int)ceil_div(p.N, p.bn);
        const int64_t tiles = (int64_t)p.tm * p.tn;
        if (tiles > (1 << 22)) return fail(RACE_E_UNSUPPORTED, "%d x %d outputs exceed one launch", p.M, p.N);
    }
    if (p.splits < 1) p.splits = 1;
    p.kper = (int)ceil_div(p.ksteps, p.splits);
    p.splits = (int)ceil_div(p.ksteps, p.kper);
    if (p.splits > 1) p.parts = align256((size_t)p.splits * p.M * p.N * sizeof(float));
    return RACE_OK;
}

template <typename TO> void launch_sum(const MatArgs &m, int splits, hipStream_t s) {
    const int64_t n = ceil_div(m.M * m.N, 1024);
    k_split_sum<TO><<<(unsigned)(n < 8192 ? n : 8192), 256, 0, s>>>(m, splits);
}

template <typename TO> void launch_tiles(const MatPlan &p, const MatArgs &m, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)p.tm * p.tn), (unsigned)p.splits);
    if constexpr (!std::is_same<TO, float>::value) {
        if (p.bm == 256) k_block_matmul<256, 256, 2, 2, TO><<<grid, 256, 0, s>>>(m);
    }
    if (p.bm == 128) k_block_matmul<128, 128, 2, 2, TO><<<grid, 256, 0, s>>>(m);
    if (p.splits > 1) launch_sum<TO>(m, p.splits, s);
}

template <typename TX, bool QUANT, typename TO>
void launch_few(const MatPlan &p, const SkinnyArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)p.tn, (unsigned)p.splits);
    if (p.M <= 16) {
        k_block_matmul_few<1, TX, QUANT, TO><<<grid, 512, 0, s>>>(a);
    } else if constexpr (!QUANT) {
        k_block_matmul_few<2, TX, false, TO><<<grid, 512, 0, s>>>(a);
    }
    if (p.splits > 1) launch_sum<TO>(a.m, p.splits, s);
}

int check_product(const race_blocks *b, int64_t rows, const float *bias, void *out, int out_dtype, int64_t out_ld,
                  const MatPlan &p, size_t codes, const void *ws, size_t ws_bytes) {
    int rc;
    if ((rc = check_rows("out", out, esize(out_dtype), rows, b->rows, out_ld, true))) return rc;
    if (bias && (rc = check_ptr("bias", bias, 4))) return rc;
    const size_t need = p.pack_a + p.pack_b + p.parts + codes;
    if (need && (!ws || ws_bytes < need)) return fail(RACE_E_WORKSPACE, "workspace %zu bytes < required %zu", ws_bytes, need);
    if (need && (uintptr_t)ws % 16) return fail(RACE_E_INVALID, "workspace is not 16-byte aligned");
    return RACE_OK;
}

// The codes of a few rows that quantise_first() wants, at ws.
struct LinearCodes {
    race_blocks a;
    size_t bytes;
};
LinearCodes linear_codes(int64_t rows, const race_blocks *b, char *ws) {
    LinearCodes q{};
    if (!quantise_first(b)) return q;
    q.a.rows = rows;
    q.a.cols = b->cols;
    q.a.ld = round_up(b->cols, 16);
    q.a.scale_ld = ceil_div(b->cols, BLK);
    q.a.block_rows = 1;
    const size_t codes = align256((size_t)(rows * q.a.ld));
    q.a.codes = ws;
    q.a.scale = ws ? ws + codes : nullptr;
    q.bytes = codes + align256((size_t)(rows * q.a.scale_ld));
    return q;
}

MatArgs mat_args(const MatPlan &p, const race_blocks *a, const race_blocks *b, const float *bias, void *out,
                 int64_t out_ld, void *ws) {
    MatArgs m{};
    m.a = (const uint8_t *)a->codes;
    m.b = (const uint8_t *)b->codes;
    m.sa = (const uint8_t *)a->scale;
    m.sb = (const uint8_t *)b->scale;
    m.bias = bias;
    m.out = out;
    m.part = p.parts ? (float *)((char *)ws + p.pack_a + p.pack_b) : nullptr;
    m.M = p.M;
    m.N = p.N;
    m.K = p.K;
    m.lda = a->ld;
    m.ldb = b->ld;
    m.lsa = a->scale_ld;
    m.lsb = b->scale_ld;
    m.ldo = out_ld;
    m.sha = a->block_rows == BLK ? 7 : 0;
    m.shb = b->block_rows == BLK ? 7 : 0;
    m.ksteps = p.ksteps;
    m.kper = p.kper;
    m.tm = p.tm;
    m.tn = p.tn;
    return m;
}

}  // namespace
}  // namespace race

using namespace race;

extern "C" {

int race_rms_norm(const race_norm_desc *d, const void *x, const void *residual, const float *w, void *y, void *h,
                  float *rstd, void *stream) {
    return norm_forward(d, x, residual, w, y, false, nullptr, 0, h, rstd, stream, "race_rms_norm");
}

int race_rms_norm_codes(const race_norm_desc *d, const void *x, const void *residual, const float *w,
                        const race_blocks *y, void *h, void *stream) {
    if (int rc = check_norm(d)) return rc;
    if (int rc = check_out_blocks("y", y)) return rc;
    if (y->rows != d->rows || y->cols != d->D || y->block_rows != 1)
        return fail(RACE_E_INVALID, "y must hold [rows][D] with a scale for every row (got %lld x %lld, %d rows a scale)",
                    (ll)y->rows, (ll)y->cols, y->block_rows);
    race_norm_desc dd = *d;
    dd.y_stride = y->ld;
    return norm_forward(&dd, x, residual, w, y->codes, true, (uint8_t *)y->scale, y->scale_ld, h, nullptr, stream,
                        "race_rms_norm_codes");
}

size_t race_rms_norm_bwd_workspace_bytes(const race_norm_desc *d) {
    if (check_norm(d)) return 0;
    ok();
    return (size_t)norm_bwd_grid(d->rows, d->D) * d->D * sizeof(float);
}

int race_rms_norm_bwd(const race_norm_desc *d, const void *x, const void *residual, const float *w, const float *rstd,
                      const void *dy, const void *dh, void *dx, void *dresidual, float *dw, void *ws, size_t ws_bytes,
                      void *stream) {
    if (int rc = check_norm(d)) return rc;
    const int ex = esize(d->dtype), er = esize(d->r_dtype);
    int rc;
    if (x && (rc = check_rows("x", x, ex, d->rows, d->D, d->x_stride, false))) return rc;
    if ((rc = check_rows("residual", residual, er, d->rows, d->D, d->r_stride, false)) || (rc = check_ptr("w", w, 4)) ||
        (rc = check_ptr("rstd", rstd, 4)) || (rc = check_rows("dy", dy, ex, d->rows, d->D, d->dy_stride, false)) ||
        (rc = check_ptr("dw", dw, 4)))
        return rc;
    if (dh && (rc = check_rows("dh", dh, er, d->rows, d->D, d->dh_stride, false))) return rc;
    if (dx && (rc = check_rows("dx", dx, ex, d->rows, d->D, d->dx_stride, true))) return rc;
    if (dresidual && (rc = check_rows("dresidual", dresidual, er, d->rows, d->D, d->dr_stride, true))) return rc;
    const int64_t grid = norm_bwd_grid(d->rows, d->D);
    const size_t need = (size_t)grid * d->D * sizeof(float);
    if (!ws || ws_bytes < need) return fail(RACE_E_WORKSPACE, "workspace %zu bytes < required %zu", ws_bytes, need);
    if ((rc = check_ptr("workspace", ws, 4))) return rc;
    NormArgs a{};
    a.x = x;
    a.r = residual;
    a.w = w;
    a.rstd_in = rstd;
    a.dy = dy;
    a.dh = dh;
    a.dx = dx;
    a.dr = dresidual;
    a.dw_part = (float *)ws;
    a.rows = d->rows;
    a.D = d->D;
    a.xs = d->x_stride;
    a.rs = d->r_stride;
    a.dys = d->dy_stride;
    a.dhs = d->dh_stride;
    a.dxs = d->dx_stride;
    a.drs = d->dr_stride;
    hipStream_t s = (hipStream_t)stream;
    norm_types(d->dtype, d->r_dtype, [&](auto tx, auto tr) {
        norm_config<16384>(d->D, [&](auto V, auto NV, auto L) {
            k_rms_norm_bwd<decltype(tx), decltype(tr), V, NV, L><<<(unsigned)grid, NORM_THREADS, 0, s>>>(a);
        });
    });
    k_column_sum<float><<<(unsigned)ceil_div(d->D, CS_COLS), 256, 0, s>>>((const float *)ws, dw, (int)grid, d->D);
    return launched("race_rms_norm_bwd");
}

size_t race_quantize_workspace_bytes(int64_t rows, int64_t cols) {
    if (rows < 1 || cols < 1) {
        fail(RACE_E_INVALID, "rows and cols must be >= 1 (got %lld, %lld)", (ll)rows, (ll)cols);
        return 0;
    }
    ok();
    return (size_t)ceil_div(rows, BLK) * cols * sizeof(float);
}

int race_quantize(const void *x, int32_t dtype, int64_t rows, int64_t cols, int64_t ld, const race_blocks *y,
                  const race_blocks *yt, float *sums, void *ws, size_t ws_bytes, void *stream) {
    int rc;
    if (!dtype_ok(dtype)) return fail(RACE_E_INVALID, "dtype %d is not RACE_DTYPE_F32 or RACE_DTYPE_BF16", dtype);
    if (rows < 1 || cols < 1) return fail(RACE_E_INVALID, "rows and cols must be >= 1 (got %lld, %lld)", (ll)rows, (ll)cols);
    if ((rc = check_rows("x", x, esize(dtype), rows, cols, ld, false))) return rc;
    if (!y && !yt) return fail(RACE_E_INVALID, "neither y nor yt is given");
    if (y && ((rc = check_out_blocks("y", y)))) return rc;
    if (yt && ((rc = check_out_blocks("yt", yt)))) return rc;
    if (y && (y->rows != rows || y->cols != cols))
        return fail(RACE_E_INVALID, "y is %lld x %lld, x %lld x %lld", (ll)y->rows, (ll)y->cols, (ll)rows, (ll)cols);
    if (yt && (yt->rows != cols || yt->cols != rows))
        return fail(RACE_E_INVALID, "yt is %lld x %lld, x %lld x %lld", (ll)yt->rows, (ll)yt->cols, (ll)rows, (ll)cols);
    if (y && yt && y->block_rows != yt->block_rows)
        return fail(RACE_E_INVALID, "y and yt have blocks of the same rows (got %d and %d)", y->block_rows, yt->block_rows);
    if (rows > ((int64_t)1 << 31) - 256 || cols > ((int64_t)1 << 31) - 256)
        return fail(RACE_E_UNSUPPORTED, "%lld x %lld exceeds 2^31 rows or columns", (ll)rows, (ll)cols);
    const int64_t tr = ceil_div(rows, BLK), tc = ceil_div(cols, BLK);
    if (sums) {
        const size_t need = (size_t)tr * cols * sizeof(float);
        if ((rc = check_ptr("sums", sums, 4))) return rc;
        if (!ws || ws_bytes < need) return fail(RACE_E_WORKSPACE, "workspace %zu bytes < required %zu", ws_bytes, need);
        if ((rc = check_ptr("workspace", ws, 4))) return rc;
    }
    QuantArgs a{};
    a.x = x;
    a.rows = rows;
    a.cols = cols;
    a.ld = ld;
    if (y) {
        a.codes = (uint8_t *)y->codes;
        a.scale = (uint8_t *)y->scale;
        a.codes_ld = y->ld;
        a.scale_ld = y->scale_ld;
    }
    if (yt) {
        a.codes_t = (uint8_t *)yt->codes;
        a.scale_t = (uint8_t *)yt->scale;
        a.codes_t_ld = yt->ld;
        a.scale_t_ld = yt->scale_ld;
    }
    a.sums = sums ? (float *)ws : nullptr;
    hipStream_t s = (hipStream_t)stream;
    const bool block = (y ? y : yt)->block_rows == BLK;
    if (y && !yt && !sums && !block) {
        const int64_t n = ceil_div(rows * tc, 16);
        const unsigned grid = (unsigned)(n < (1 << 20) ? n : 1 << 20);
        if (dtype == RACE_DTYPE_BF16) k_quantize_rows<bf16><<<grid, 256, 0, s>>>(a);
        else k_quantize_rows<float><<<grid, 256, 0, s>>>(a);
        return launched("race_quantize");
    }
    if (tr > 65535 || tr * tc > (1 << 24) - 1)
        return fail(RACE_E_UNSUPPORTED, "%lld x %lld exceeds one launch's tiles", (ll)rows, (ll)cols);
    const dim3 grid((unsigned)tc, (unsigned)tr);
    if (dtype == RACE_DTYPE_BF16) {
        if (block) k_quantize_tile<bf16, true><<<grid, 256, 0, s>>>(a);
        else k_quantize_tile<bf16, false><<<grid, 256, 0, s>>>(a);
    } else {
        if (block) k_quantize_tile<float, true><<<grid, 256, 0, s>>>(a);
        else k_quantize_tile<float, false><<<grid, 256, 0, s>>>(a);
    }
    if (sums) k_column_sum<float><<<(unsigned)ceil_div(cols, CS_COLS), 256, 0, s>>>(a.sums, sums, (int)tr, cols);
    return launched("race_quantize");
}

size_t race_block_matmul_workspace_bytes(const race_blocks *a, const race_blocks *b, int32_t out_dtype) {
    MatPlan p;
    if (mat_plan(a, b, out_dtype, p)) return 0;
    ok();
    return p.pack_a + p.pack_b + p.parts;
}

int race_block_matmul(const race_blocks *a, const race_blocks *b, const float *bias, void *out, int32_t out_dtype,
                      int64_t out_ld, void *ws, size_t ws_bytes, void *stream) {
    MatPlan p;
    int rc;
    if ((rc = mat_plan(a, b, out_dtype, p)) || (rc = check_product(b, a->rows, bias, out, out_dtype, out_ld, p, 0, ws, ws_bytes)))
        return rc;
    SkinnyArgs sk{};
    MatArgs &m = sk.m;
    m = mat_args(p, a, b, bias, out, out_ld, ws);
    hipStream_t s = (hipStream_t)stream;
    if (p.few) {
        if (out_dtype == RACE_DTYPE_BF16) launch_few<bf16, false, bf16>(p, sk, s);
        else launch_few<bf16, false, float>(p, sk, s);
        return launched("race_block_matmul");
    }
    if (p.pack_a || p.pack_b) {
        RepackArgs r{};
        r.cols = a->cols;
        r.y_ld = p.K;
        auto add = [&](int i, const race_blocks *x, void *to) {
            r.x[i] = (const uint8_t *)x->codes;
            r.y[i] = (uint8_t *)to;
            r.rows[i] = x->rows;
            r.ld[i] = x->ld;
        };
        if (p.pack_a) {
            add(0, a, ws);
            m.a = r.y[0];
            m.lda = p.K;
        }
        if (p.pack_b) {
            add(1, b, (char *)ws + p.pack_a);
            m.b = r.y[1];
            m.ldb = p.K;
        }
        const int64_t n = ceil_div((r.rows[0] + r.rows[1]) * (p.K / 16), 256);
        k_repack<<<(unsigned)(n < 65536 ? n : 65536), 256, 0, s>>>(r);
    }
    if (out_dtype == RACE_DTYPE_BF16) launch_tiles<bf16>(p, m, s);
    else launch_tiles<float>(p, m, s);
    return launched("race_block_matmul");
}

int64_t race_block_linear_rows(void) { return kLinearRows; }

size_t race_block_linear_workspace_bytes(int64_t rows, const race_blocks *b, int32_t out_dtype) {
    if (!b || rows < 1 || rows > kLinearRows) {
        fail(RACE_E_INVALID, "1 to %d rows (got %lld) and a matrix b", kLinearRows, (ll)rows);
        return 0;
    }
    MatPlan p;
    race_blocks a = *b;
    a.rows = rows;
    if (mat_plan(&a, b, out_dtype, p)) return 0;
    ok();
    return p.parts + linear_codes(rows, b, nullptr).bytes;
}

int race_block_linear(const void *x, int32_t dtype, int64_t rows, int64_t x_ld, const race_blocks *b, const float *bias,
                      void *out, int32_t out_dtype, int64_t out_ld, void *ws, size_t ws_bytes, void *stream) {
    int rc;
    if (!dtype_ok(dtype)) return fail(RACE_E_INVALID, "dtype %d is not RACE_DTYPE_F32 or RACE_DTYPE_BF16", dtype);
    if (rows < 1 || rows > kLinearRows)
        return fail(RACE_E_UNSUPPORTED, "rows=%lld: 1 to %d (quantise more rows first)", (ll)rows, kLinearRows);
    if ((rc = check_blocks("b", b))) return rc;
    if ((rc = check_rows("x", x, esize(dtype), rows, b->cols, x_ld, false))) return rc;
    race_blocks a = *b;  // sizes alone: x takes its codes' place
    a.rows = rows;
    MatPlan p;
    if ((rc = mat_plan(&a, b, out_dtype, p)) ||
        (rc = check_product(b, rows, bias, out, out_dtype, out_ld, p, linear_codes(rows, b, nullptr).bytes, ws, ws_bytes)))
        return rc;
    const LinearCodes q = linear_codes(rows, b, (char *)ws + p.parts);
    if (q.bytes) {
        if ((rc = race_quantize(x, dtype, rows, b->cols, x_ld, &q.a, nullptr, nullptr, nullptr, 0, stream))) return rc;
        a = q.a;
    }
    SkinnyArgs sk{};
    sk.m = mat_args(p, &a, b, bias, out, out_ld, ws);
    sk.x = x;
    sk.ldx = x_ld;
    hipStream_t s = (hipStream_t)stream;
    const bool f32 = out_dtype == RACE_DTYPE_F32;
    if (q.bytes) f32 ? launch_few<bf16, false, float>(p, sk, s) : launch_few<bf16, false, bf16>(p, sk, s);
    else if (dtype == RACE_DTYPE_BF16) f32 ? launch_few<bf16, true, float>(p, sk, s) : launch_few<bf16, true, bf16>(p, sk, s);
    else f32 ? launch_few<float, true, float>(p, sk, s) : launch_few<float, true, bf16>(p, sk, s);
    return launched("race_block_linear");
}

int race_adamw(const race_adamw_desc *d, const race_adamw_tensor *t, int64_t count, void *stream) {
    if (!d) return fail(RACE_E_INVALID, "descriptor is NULL");
    if (!dtype_ok(d->p_dtype) || !dtype_ok(d->g_dtype))
        return fail(RACE_E_INVALID, "dtype %d or %d is not RACE_DTYPE_F32 or RACE_DTYPE_BF16", d->p_dtype, d->g_dtype);
    if (d->bits != 32 && d->bits != 8) return fail(RACE_E_INVALID, "states have 32 or 8 bits (got %d)", d->bits);
    if (!(d->beta_m >= 0 && d->beta_m < 1) || !(d->beta_v >= 0 && d->beta_v < 1))
        return fail(RACE_E_INVALID, "betas must be in [0, 1) (got %g, %g)", d->beta_m, d->beta_v);
    if (!std::isfinite(d->lr) || !std::isfinite(d->weight_decay) || !(d->eps >= 0) || !std::isfinite(d->eps))
        return fail(RACE_E_INVALID, "lr, weight_decay and eps must be finite, eps >= 0");
    if (!d->step_ptr && !(d->step >= 1)) return fail(RACE_E_INVALID, "step must be >= 1 (got %g)", d->step);
    if (d->step_ptr && (uintptr_t)d->step_ptr % 4) return fail(RACE_E_INVALID, "step_ptr is not 4-byte aligned");
    if (count < 0 || (count && !t)) return fail(RACE_E_INVALID, "count=%lld tensors", (ll)count);
    const bool eight = d->bits == 8;
    for (int64_t i = 0; i < count; ++i) {
        int rc;
        if (t[i].n < 0) return fail(RACE_E_INVALID, "tensor %lld has %lld elements", (ll)i, (ll)t[i].n);
        if (t[i].n == 0) continue;
        if (t[i].n > ((int64_t)1 << 35)) return fail(RACE_E_UNSUPPORTED, "tensor %lld has %lld elements (at most 2^35)", (ll)i, (ll)t[i].n);
        if ((rc = check_ptr("p", t[i].p, esize(d->p_dtype))) || (rc = check_ptr("g", t[i].g, esize(d->g_dtype))) ||
            (rc = check_ptr("m", t[i].m, eight ? 1 : 4)) || (rc = check_ptr("v", t[i].v, eight ? 1 : 4)))
            return rc;
        if (eight && ((rc = check_ptr("m_scale", t[i].m_scale, 1)) || (rc = check_ptr("v_scale", t[i].v_scale, 1)))) return rc;
    }
    AdamArgs a{};
    a.seed = d->seed;
    a.mixed_seed = mix32(d->seed);
    a.b1 = (float)d->beta_m;
    a.c1 = (float)(1.0 - d->beta_m);
    a.b2 = (float)d->beta_v;
    a.c2 = (float)(1.0 - d->beta_v);
    a.keep = (float)(1.0 - d->lr * d->weight_decay);
    a.eps = (float)d->eps;
    a.lr = d->lr;
    a.db1 = d->beta_m;
    a.db2 = d->beta_v;
    a.step = d->step_ptr;
    if (!a.step) {
        a.lr_bc1 = (float)(d->lr / (1.0 - std::pow(d->beta_m, d->step)));
        a.inv_root_bc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(d->beta_v, d->step)));
    }
    hipStream_t s = (hipStream_t)stream;
    int64_t place = 0;
    uint32_t blocks = 0;
    bool any = false;
    auto flush = [&] {
        if (!a.count) return;
        any = true;
        const bool pb = d->p_dtype == RACE_DTYPE_BF16, gb = d->g_dtype == RACE_DTYPE_BF16;
        auto go = [&](auto tp, auto tg) {
            if (eight) k_adamw<decltype(tp), decltype(tg), true><<<blocks, ADAM_THREADS, 0, s>>>(a);
            else k_adamw<decltype(tp), decltype(tg), false><<<blocks, ADAM_THREADS, 0, s>>>(a);
        };
        if (pb && gb) go(bf16{}, bf16{});
        else if (pb) go(bf16{}, float{});
        else if (gb) go(float{}, bf16{});
        else go(float{}, float{});
        a.count = 0;
        blocks = 0;
    };
    for (int64_t i = 0; i < count; ++i) {
        if (t[i].n == 0) continue;
        const int64_t nb = ceil_div(t[i].n, ADAM_CHUNK);
        if (a.count == ADAM_TENSORS || (int64_t)blocks + nb >= (1 << 24)) flush();  // 2^32 work-items a launch
        const int k = a.count++;
        a.p[k] = t[i].p;
        a.g[k] = t[i].g;
        a.m[k] = t[i].m;
        a.v[k] = t[i].v;
        a.ms[k] = (uint8_t *)t[i].m_scale;
        a.vs[k] = (uint8_t *)t[i].v_scale;
        a.n[k] = t[i].n;
        a.first[k] = blocks;
        a.place[k] = (uint32_t)place;
        blocks += (uint32_t)nb;
        place += round_up(t[i].n, BLK);
    }
    flush();
    return any ? launched("race_adamw") : ok();
}

}  // extern "C"
