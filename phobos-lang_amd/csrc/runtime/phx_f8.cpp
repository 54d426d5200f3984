// Entry points of the operators over 8-bit rows and weights: the norm, the gated
// activation, products.  Arguments are checked here; what lies in device memory
// (groups' starts, lists of rows) the kernels check themselves (gemm_f8.hip).
#include <algorithm>
#include <cmath>
#include <iterator>

#include "../kernels/phx_f8.h"
#include "phx_internal.h"

using namespace phx;

namespace {

const char *const kRowsFile = "f8_rows.hsaco";
const char *const kGemmFile = "gemm_f8.hsaco";

// (file and entry are literals: aux_function knows them by address)
int launch(const char *file, const char *entry, int64_t groups, uint32_t threads, hipStream_t s,
           void *record) {
    hipFunction_t f;
    if (int rc = aux_function(file, entry, &f)) return rc;
    void *args[] = {record};
    hipError_t e = hipModuleLaunchKernel(f, (uint32_t)groups, 1, 1, threads, 1, 1, 0, s, args,
                                         nullptr);
    return e == hipSuccess ? PHX_OK : hip_error(e, entry);
}

bool known(phx_dtype t) { return t == PHX_F32 || t == PHX_F16; }
int64_t size_of(phx_dtype t) { return t == PHX_F16 ? 2 : 4; }
int64_t blocks_of(int64_t k) { return (k + PHX_F8_BLOCK - 1) / PHX_F8_BLOCK; }

constexpr int64_t kMost = INT64_C(1) << 40;   // of a stride: products with 2^22 rows stay in 64 bits
constexpr int64_t kMostRows = INT32_MAX;
constexpr int64_t kMostThreads = UINT32_MAX;  // of a launch along one axis
constexpr int64_t kMostK = 1 << 22;           // 256 rows of it are within 32-bit offsets

constexpr int64_t kMostScales = 1 << 20;      // and 256 rows of these

// 8-bit rows, with their strides filled in.
int check_f8(const phx_f8_rows *r, phx_f8_rows *out, const char *who) {
    if (!r) return set_error(PHX_E_INVALID, "%s: null rows", who);
    *out = *r;
    if (r->rows < 0 || r->rows > kMostRows || r->k < 16 || r->k % 16 || r->k > kMostK)
        return set_error(PHX_E_INVALID,
                         "%s: 8-bit rows need 0 .. 2^31-1 rows of K elements, 16 <= K <= %lld with "
                         "K%%16==0 (got %lld of %lld)",
                         who, (long long)kMostK, (long long)r->rows, (long long)r->k);
    const int64_t blocks = blocks_of(r->k);
    if (!out->ld) out->ld = r->k;
    if (!out->lds) out->lds = (blocks + 3) / 4 * 4;
    if (out->ld < r->k || out->ld % 16 || out->ld > kMostK || out->lds < blocks || out->lds % 4 ||
        out->lds > kMostScales)
        return set_error(PHX_E_INVALID,
                         "%s: 8-bit rows must be at least K apart, in whole 16 bytes, and their scales "
                         "at least ceil(K/128), in fours (got %lld, %lld)",
                         who, (long long)r->ld, (long long)r->lds);
    if (r->rows && (!r->codes || !r->scales || ((r->codes | r->scales) & 15)))
        return set_error(PHX_E_INVALID, "%s: codes and scales must be 16-byte aligned", who);
    return PHX_OK;
}

// Rows of `width` elements of type t, `ld` apart (0: dense).
int check_rows(phx_dtype t, uint64_t ptr, int64_t width, int64_t *ld, const char *who,
               const char *what) {
    if (!*ld) *ld = width;
    if (*ld < width || *ld > kMost || *ld * size_of(t) % 16)
        return set_error(PHX_E_INVALID, "%s: rows of %s must be at least %lld elements apart, in "
                         "whole 16-byte chunks (got %lld)", who, what, (long long)width,
                         (long long)*ld);
    if (!ptr || (ptr & 15))
        return set_error(PHX_E_INVALID, "%s: %s must be 16-byte aligned", who, what);
    return PHX_OK;
}

// ------------------------------------------------------------------ the norm
// How a norm runs: up to 64 chunks of 16 bytes a row by as many lanes, a power of two
// (781250 rows of 128, f16, with the sum: 124 us, by a wave each 335); up to 128 by a
// wave (16384 rows of 1024, f16: 26.9 us, by 128 threads of a workgroup of their own
// 32.1); more by a workgroup of as many threads as one, two, four or eight chunks each
// take: two from 512 on (8192 rows of 8192, f16: 87 us, four 95; 4096 of 4096, f32:
// 42.8 us, four 47.3).
struct NormForm {
    int64_t rows;  // of a workgroup
    uint32_t threads;
    const char *entry;
};

NormForm norm_form(phx_dtype t, int64_t K) {
    static const char *const names[2][6] = {
        {"norm_f8_rows_f16_c1", "norm_f8_rows_f16_c2", "norm_f8_f16_c1", "norm_f8_f16_c2",
         "norm_f8_f16_c4", nullptr},
        {"norm_f8_rows_f32_c1", "norm_f8_rows_f32_c2", "norm_f8_f32_c1", "norm_f8_f32_c2",
         "norm_f8_f32_c4", "norm_f8_f32_c8"}};
    const char *const *name = names[t == PHX_F16 ? 0 : 1];
    const int64_t chunks = K * size_of(t) / 16;
    int64_t lanes = 2;
    while (lanes < chunks && lanes < 64) lanes *= 2;
    if (chunks <= 128) return {256 / lanes, 256, name[chunks > 64]};
    const int64_t of_thread = chunks <= 512 ? 1 : chunks <= 2048 ? 2 : chunks <= 4096 ? 4 : 8;
    const int64_t threads = (chunks + of_thread - 1) / of_thread;
    return {1, (uint32_t)((threads + 63) / 64 * 64),
            name[of_thread == 1 ? 2 : of_thread == 2 ? 3 : of_thread == 4 ? 4 : 5]};
}

// ------------------------------------------------------------------ products
// A kernel of gemm_f8.hip: the columns and rows of a workgroup, how many blocks of K
// it takes in a step, and how many workgroups a CU holds.  What it is weighed by: `step`
// for each step, or `shared` for every workgroup of the CU where that is more, and `rest`
// for what is before and behind the steps.  The constants are fitted to which kernel is
// the fastest over 502 shapes a type (1 to 4096 rows, K 64 to 8192; grouped: 1 to 512 rows
// each of 5 to 61 experts), not to its time: that is 1.1 to 4.1 times the sum in ns for
// f16, half of the shapes above 2.1, and 0.65 to 5.3 times, above 1.6, for f32.
struct GemmForm {
    int64_t columns, rows, blocks;
    uint32_t threads;
    int64_t held, step, shared, rest;
    const char *entry;
};
#define FORM(t, wn, wm, nt, mt, wk, st, held, step, shared, rest)                 \
    {16 * wn * nt, 16 * wm * mt, wk, 64 * wn * wm * wk, held, step, shared, rest, \
     "gemm_f8_" #t "_" #wn "x" #wm "_" #nt "x" #mt "_k" #wk "_s" #st}
const GemmForm kGemmF16[] = {FORM(f16, 1, 1, 2, 1, 4, 4, 1, 191, 4, 2331),
                             FORM(f16, 1, 1, 2, 1, 4, 2, 3, 0, 298, 1650),
                             FORM(f16, 2, 1, 2, 1, 4, 3, 1, 498, 0, 1519),
                             FORM(f16, 2, 1, 2, 2, 2, 3, 2, 0, 277, 1629),
                             FORM(f16, 2, 2, 2, 2, 2, 4, 1, 372, 73, 1515),
                             FORM(f16, 2, 2, 2, 2, 1, 4, 2, 190, 146, 1495),
                             FORM(f16, 2, 2, 4, 2, 1, 3, 2, 380, 255, 1306),
                             FORM(f16, 2, 4, 8, 2, 1, 3, 1, 552, 3, 1567),
                             FORM(f16, 2, 4, 8, 4, 1, 2, 1, 939, 2, 2173)};
const GemmForm kGemmF32[] = {FORM(f32, 1, 1, 2, 1, 4, 2, 3, 930, 402, 950),
                             FORM(f32, 1, 1, 2, 1, 8, 3, 1, 1450, 0, 2300),
                             FORM(f32, 2, 1, 2, 2, 2, 3, 2, 649, 441, 1079),
                             FORM(f32, 1, 2, 4, 2, 4, 2, 1, 1358, 0, 1512),
                             FORM(f32, 2, 2, 2, 2, 1, 4, 2, 455, 332, 1018),
                             FORM(f32, 2, 2, 4, 2, 1, 3, 2, 780, 478, 889),
                             FORM(f32, 2, 2, 4, 4, 1, 2, 2, 1209, 774, 751)};
#undef FORM

// (in 64-bit floating point: sizes that are refused later would overflow; a weight, no time)
double estimate(const GemmForm &f, int64_t M, int64_t N, int64_t K, int64_t experts) {
    // (which experts have how many rows is not known here: all have some)
    const int64_t live = std::min(experts, M);
    const int64_t tiles = experts == 1 ? (M + f.rows - 1) / f.rows
                                       : std::max(live, M / f.rows + live / 2);
    const int64_t groups = tiles * ((N + f.columns - 1) / f.columns);
    const int64_t steps = (blocks_of(K) + f.blocks - 1) / f.blocks, round = 256 * f.held;
    auto of = [&](int64_t each) { return steps * std::max(f.step, each * f.shared) + f.rest; };
    const int64_t left = groups % round;
    return (double)(groups / round) * of(f.held) + (left ? of((left + 255) / 256) : 0);
}

// The kernel that weighs least. Over those shapes its time is 1.013 (f16) and 1.007
// (f32) times that of the fastest one, at most 1.32 and 1.27 times; any one kernel for
// all is 1.24 times and more. (Columns x rows; f16.) 8192 x 16384 x 8192: 256 x 256
// 922 us, 256 x 128 1058; 384 x 16384 x 8192: 256 x 128 70 us, 256 x 256 100; 1 x 4096
// x 4096: 32 x 16 with four stages 6.4 us, with two 8.2, 64 x 64 9.5, 256 x 256 30; 64 x
// 16384 x 8192: 64 x 64 over two blocks 29.4 us, over one 30.5, 64 x 32 36.7. Not the
// fastest: 257 x 8192 x 8192, 64 x 64 43.8 us, 128 x 64 38.3; 1 x 16384 x 8192, 64 x 16
// 25.5 us, 32 x 16 with two stages 24.8.
const GemmForm &gemm_form(phx_dtype t, int64_t M, int64_t N, int64_t K, int64_t experts) {
    const GemmForm *first = t == PHX_F16 ? std::begin(kGemmF16) : std::begin(kGemmF32);
    const GemmForm *last = t == PHX_F16 ? std::end(kGemmF16) : std::end(kGemmF32);
    const GemmForm *best = first;
    double least = INFINITY;
    for (; first != last; ++first) {
        const double w = estimate(*first, M, N, K, experts);
        if (w < least) best = first, least = w;
    }
    return *best;
}

int product(phx_stream s, const phx_f8_rows *a, const phx_f8_weights *w, bool grouped,
            uint64_t starts, uint64_t list, int64_t M, phx_dtype t, uint64_t c, float alpha,
            float beta, int64_t ldc, const char *who) {
    phx_f8_rows r;
    if (!known(t)) return set_error(PHX_E_INVALID, "%s: unknown type %d", who, (int)t);
    if (int rc = check_f8(a, &r, who)) return rc;
    if (!w) return set_error(PHX_E_INVALID, "%s: null weights", who);
    if (w->n < 1 || w->n > kMostRows || w->k != r.k || w->experts < 1 || w->experts > 65535)
        return set_error(PHX_E_INVALID,
                         "%s: weights of 1 .. 65535 experts, N > 0 and the rows' K (got %lld of %lld "
                         "x %lld, rows of %lld)",
                         who, (long long)w->experts, (long long)w->n, (long long)w->k,
                         (long long)r.k);
    if (!grouped && w->experts != 1)
        return set_error(PHX_E_INVALID, "%s: %lld experts take a grouped product", who,
                         (long long)w->experts);
    if (!grouped) M = r.rows;
    if (M < 0 || M > kMostRows)
        return set_error(PHX_E_INVALID, "%s: %lld rows", who, (long long)M);
    if (grouped && !list && M > r.rows)
        return set_error(PHX_E_INVALID, "%s: %lld rows of C, %lld of A", who, (long long)M,
                         (long long)r.rows);
    if (list && (r.rows * r.ld > INT32_MAX || r.rows * r.lds * 4 > INT32_MAX))
        return set_error(PHX_E_INVALID, "%s: with a list A's codes and scales are below 2 GiB (%lld rows "
                         "%lld apart)", who, (long long)r.rows, (long long)r.ld);
    if (!ldc) ldc = w->n;
    if (ldc < w->n || ldc > kMost)
        return set_error(PHX_E_INVALID, "%s: rows of C must be at least N apart (got %lld)", who,
                         (long long)ldc);
    if (M && (!w->codes || !w->scales || !c || (w->codes & 15) || (w->scales & 3) ||
              (c & (size_of(t) - 1))))
        return set_error(PHX_E_INVALID, "%s: weights' codes must be 16-byte aligned, their scales and "
                         "C by element", who);
    if (M && grouped && (!starts || ((starts | list) & 3)))
        return set_error(PHX_E_INVALID, "%s: starts and list are i32 arrays", who);
    const GemmForm &f = gemm_form(t, M, w->n, r.k, w->experts);
    // (groups of rows: each that has any has a first tile, and only whole tiles behind it add
    // one; workgroups behind what there is read the starts and end)
    const int64_t live = std::min(grouped ? w->experts : 1, M);
    const int64_t tiles = (live + (M - live) / f.rows) * ((w->n + f.columns - 1) / f.columns);
    if (tiles > kMostThreads / f.threads)
        return set_error(PHX_E_INVALID, "%s: %lld x %lld is too large", who, (long long)M,
                         (long long)w->n);
    if (int rc = on_device((hipStream_t)s)) return rc;
    if (!M) return PHX_OK;
    PhxF8Gemm p = {r.codes, r.scales, w->codes, w->scales, c, starts, list, M, w->n, r.k, r.rows,
                   r.ld, r.lds, ldc, w->experts, alpha, beta};
    return launch(kGemmFile, f.entry, tiles, f.threads, (hipStream_t)s, &p);
}

}  // namespace

extern "C" {

int phx_norm_f8(phx_stream s, phx_dtype t, uint64_t x, uint64_t r, uint64_t gain, uint64_t h,
                uint64_t y, const phx_f8_rows *q, int64_t M, int64_t K, float eps, int64_t ldx,
                int64_t ldr, int64_t ldh, int64_t ldy) {
    const char *who = "norm_f8";
    if (!known(t)) return set_error(PHX_E_INVALID, "%s: unknown type %d", who, (int)t);
    if (M < 0 || M > kMostRows || K < 16 || K % 16 || K > PHX_F8_NORM_MOST)
        return set_error(PHX_E_INVALID, "%s needs 0 .. 2^31-1 rows of K elements, 16 <= K <= %d with "
                         "K%%16==0 (got %lld of %lld)",
                         who, PHX_F8_NORM_MOST, (long long)M, (long long)K);
    if (!(eps >= 0.0f) || std::isinf(eps))
        return set_error(PHX_E_INVALID, "%s: eps %g", who, (double)eps);
    phx_f8_rows o = {};
    if (q) {
        if (int rc = check_f8(q, &o, who)) return rc;
        if (q->rows != M || q->k != K)
            return set_error(PHX_E_INVALID, "%s: %lld rows of %lld, 8-bit rows %lld of %lld", who,
                             (long long)M, (long long)K, (long long)q->rows, (long long)q->k);
    }
    if (M) {
        if (int rc = check_rows(t, x, K, &ldx, who, "X")) return rc;
        if (r)
            if (int rc = check_rows(t, r, K, &ldr, who, "R")) return rc;
        if (h)
            if (int rc = check_rows(t, h, K, &ldh, who, "H")) return rc;
        if (y)
            if (int rc = check_rows(t, y, K, &ldy, who, "Y")) return rc;
        if (!gain || (gain & 15))
            return set_error(PHX_E_INVALID, "%s: the gain must be 16-byte aligned", who);
        if (!y && !q) return set_error(PHX_E_INVALID, "%s: neither Y nor 8-bit rows", who);
    }
    const NormForm f = norm_form(t, K);
    const int64_t groups = (M + f.rows - 1) / f.rows;
    if (groups > kMostThreads / f.threads)
        return set_error(PHX_E_INVALID, "%s: %lld rows are too many", who, (long long)M);
    if (int rc = on_device((hipStream_t)s)) return rc;
    if (!M) return PHX_OK;
    PhxF8Rows p = {x, r, gain, h, y, o.codes, o.scales, M, K, ldx, ldr, ldh, ldy, o.ld, o.lds, 1.0 / (double)K, eps};
    return launch(kRowsFile, f.entry, groups, f.threads, (hipStream_t)s, &p);
}

int phx_glu_f8(phx_stream s, phx_dtype t, uint64_t u, const phx_f8_rows *q, int64_t ldu) {
    const char *who = "glu_f8";
    if (!known(t)) return set_error(PHX_E_INVALID, "%s: unknown type %d", who, (int)t);
    phx_f8_rows o;
    if (int rc = check_f8(q, &o, who)) return rc;
    if (o.rows)
        if (int rc = check_rows(t, u, 2 * o.k, &ldu, who, "U")) return rc;
    const int64_t per = 2 * size_of(t) == 4 ? 16 : 8;  // blocks of a workgroup
    const int64_t groups = (o.rows * blocks_of(o.k) + per - 1) / per;
    if (groups > kMostThreads / 256)
        return set_error(PHX_E_INVALID, "%s: %lld rows of %lld are too many", who, (long long)o.rows,
                         (long long)o.k);
    if (int rc = on_device((hipStream_t)s)) return rc;
    if (!o.rows) return PHX_OK;
    PhxF8Rows p = {u, 0, 0, 0, 0, o.codes, o.scales, o.rows, o.k, ldu, 0, 0, 0, o.ld, o.lds, 0.0, 0.0f};
    return launch(kRowsFile, t == PHX_F16 ? "glu_f8_f16" : "glu_f8_f32", groups, 256, (hipStream_t)s,
                  &p);
}

int phx_gemm_f8(phx_stream s, const phx_f8_rows *a, const phx_f8_weights *w, phx_dtype t, uint64_t c,
                float alpha, float beta, int64_t ldc) {
    return product(s, a, w, false, 0, 0, 0, t, c, alpha, beta, ldc, "gemm_f8");
}

int phx_gemm_f8_grouped(phx_stream s, const phx_f8_rows *a, const phx_f8_weights *w,
                        uint64_t starts, uint64_t list, int64_t M, phx_dtype t, uint64_t c,
                        float alpha, float beta, int64_t ldc) {
    return product(s, a, w, true, starts, list, M, t, c, alpha, beta, ldc, "gemm_f8_grouped");
}

}  // extern "C"
