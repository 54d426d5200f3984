// Entry points of the decode operators: products with 4-bit weights, the 4-bit
// paged cache and attention over it, copies of pages.  Arguments are checked
// here; what lies in device memory (lengths, tables, row starts) the kernels
// check themselves (kv4.hip).
#include <algorithm>
#include <exception>
#include <mutex>
#include <vector>

#include "../kernels/phx_decode.h"
#include "phx_internal.h"

using namespace phx;

namespace {

const char *const kW4File = "gemv_w4.hsaco";
const char *const kKv4File = "kv4.hsaco";
const char *const kAttendFile = "kv4_attend.hsaco";
const char *const kPagesFile = "pages.hsaco";

// (file and entry are literals: aux_function knows them by address)
int launch(const char *file, const char *entry, dim3 grid, uint32_t threads, hipStream_t s,
           void *record) {
    hipFunction_t f;
    if (int rc = aux_function(file, entry, &f)) return rc;
    void *args[] = {record};
    hipError_t e = hipModuleLaunchKernel(f, grid.x, grid.y, grid.z, threads, 1, 1, 0, s, args,
                                         nullptr);
    return e == hipSuccess ? PHX_OK : hip_error(e, entry);
}

bool known(phx_dtype t) { return t == PHX_F32 || t == PHX_F16; }
int64_t size_of(phx_dtype t) { return t == PHX_F16 ? 2 : 4; }

constexpr int64_t kMost = INT64_C(1) << 40;  // of any extent: products of two stay in 64 bits
constexpr int64_t kMostThreads = UINT32_MAX;  // of a launch along one axis
bool extent(int64_t v) { return v >= 0 && v <= INT32_MAX; }

// ------------------------------------------------------------------ 4-bit weights
// A kernel of gemv_w4.hip: the columns and rows of a workgroup, and the blocks
// of 128 k it takes at a time, in so many nanoseconds (measured; 0: only up to 16
// rows).
struct W4Form {
    int64_t columns, rows;
    uint32_t threads;
    int64_t blocks, ns;
    const char *entry[3];  // groups of 128, 64 and 32
};
#define GROUPS(name) {name "_g1", name "_g2", name "_g4"}
const W4Form kW4F16[] = {{16, 16, 512, 8, 670, GROUPS("gemv_w4_f16_n1_w8")},
                         {16, 16, 1024, 16, 1150, GROUPS("gemv_w4_f16_n1_w16")},
                         {64, 16, 512, 8, 0, GROUPS("gemv_w4_f16_n4_w8")},
                         {64, 64, 1024, 4, 1600, GROUPS("gemm_w4_f16_m4_4x4")},
                         {64, 32, 1024, 4, 1050, GROUPS("gemm_w4_f16_m2_4x4")},
                         {32, 32, 1024, 8, 1300, GROUPS("gemm_w4_f16_m2_2x8")}};
const W4Form kW4F32[] = {{16, 16, 768, 12, 2000, GROUPS("gemv_w4_f32_n1_w12")},
                         {32, 16, 768, 12, 0, GROUPS("gemv_w4_f32_n2_w12")},
                         {64, 16, 512, 8, 0, GROUPS("gemv_w4_f32_n4_w8")},
                         {256, 64, 1024, 1, 2700, GROUPS("gemm_w4_f32_m4_16x1")},
                         {128, 32, 1024, 2, 2100, GROUPS("gemm_w4_f32_m2_8x2")},
                         {64, 32, 512, 2, 1600, GROUPS("gemm_w4_f32_m2_4x2")}};
#undef GROUPS

// The kernel for a product, and the K chunks it runs in, at most `most`.
//   Up to 16 rows: 16 columns a workgroup while the CUs are not all several
// times occupied, in f16 with 16 waves over long K (4096 x 16384: 9.3 us against
// 10.6 with 8), in f32 with the 12 whose rows LDS holds (16.9 us against 18.9 with
// 8), else 64 columns (16 rows, 16384 x 8192: f16 19.5 us against 21.7,
// f32 35.0 against 61.7), in f32 32 between (8192 x 4096: 13.3 us, 16 columns 19.0,
// 64 19.1).
//   More: the one that is estimated fastest: its rounds of workgroups on the
// CUs, each K chunk's blocks; a split in 2 or 4 chunks costs its reduction
// (64 x 4096 x 16384: f16 20.9 us in 4 on tiles of 64 x 64, 24.5 in none on 32 x 32;
// 64 x 16384 x 8192: f32 60.8 in 4 on 256 x 64, 73.2 in none on 128 x 32).  Tiles of
// 16 rows that share nothing are taken while each has a CU of its own (64 x 1000
// x 4136: f16 6.6 us against 9.3, f32 11.7 against 14.0; 48 x 4096 x 4096 f16, on 768
// of them, 15.2 against 11.5).
const W4Form &w4_form(phx_dtype t, int64_t M, int64_t N, int64_t K, int64_t most,
                      int64_t *splits) {
    const W4Form *forms = t == PHX_F16 ? kW4F16 : kW4F32;
    const int64_t tiles = (N + 15) / 16;
    *splits = 1;
    if (M <= 16) {
        if (t == PHX_F32) return forms[tiles > 512 ? 2 : tiles > 256 ? 1 : 0];
        return forms[tiles >= 1024 ? 2 : tiles <= 256 && K >= 8192 ? 1 : 0];
    }
    const W4Form *best = nullptr;
    int64_t least = 0;
    for (int i = 0; i < 6; ++i) {
        const W4Form &f = forms[i];
        if (!f.ns) continue;
        const bool shared = f.rows > 16;  // the others have no split
        for (int64_t sp = 1; sp <= (shared ? 4 : 1) && sp <= std::max<int64_t>(most, 1); sp *= 2) {
            const int64_t groups =
                ((N + f.columns - 1) / f.columns) * ((M + f.rows - 1) / f.rows) * sp;
            if (!shared && groups > 256) break;
            const int64_t blocks = ((K + 127) / 128 + sp - 1) / sp;
            int64_t ns = (groups + 255) / 256 * ((blocks + f.blocks - 1) / f.blocks) * f.ns;
            if (sp > 1) ns += 3300 + (sp + 1) * M * N / 1000;
            if (!best || ns < least) {
                best = &f;
                least = ns;
                *splits = sp;
            }
        }
    }
    return *best;
}

// ------------------------------------------------------------------ 4-bit cache
int check_cache(const phx_kv4_cache *c, const char *who) {
    if (!c) return set_error(PHX_E_INVALID, "%s: null cache", who);
    if (!phx_kv4_page_bytes(c->heads, c->head_dim, c->page_tokens))
        return set_error(PHX_E_INVALID,
                         "%s: needs 1 .. 1024 heads of 64 or 128 and pages of 32, 64, 128 or 256 "
                         "tokens (got %d of %d, %d)",
                         who, c->heads, c->head_dim, c->page_tokens);
    if (c->pages < 1 || !extent(c->pages))
        return set_error(PHX_E_INVALID, "%s: pool of %lld pages", who, (long long)c->pages);
    if (!c->pool || (c->pool & 255))
        return set_error(PHX_E_INVALID, "%s: the pool must be 256-byte aligned", who);
    return PHX_OK;
}

bool has_work(const phx_kv4_batch *b) { return b->batch && b->max_q && b->rows; }

int check_batch(const phx_kv4_batch *b, const char *who) {
    if (!b) return set_error(PHX_E_INVALID, "%s: null batch", who);
    if (b->batch < 0 || b->batch > 65535)
        return set_error(PHX_E_INVALID, "%s: %lld sequences, takes 0 .. 65535", who,
                         (long long)b->batch);
    if (!extent(b->max_q) || !extent(b->rows) || !extent(b->table_stride) || !extent(b->max_len))
        return set_error(PHX_E_INVALID,
                         "%s: max_q, rows, table_stride and max_len must be 0 .. 2^31-1", who);
    if (!has_work(b)) return PHX_OK;
    if (!b->lens || (b->lens & 3) || (b->q_starts & 3) || (b->table & 3) ||
        (!b->table && b->table_stride))
        return set_error(PHX_E_INVALID, "%s: table, lens and q_starts are i32 arrays", who);
    return PHX_OK;
}

// Token rows of `heads` heads, `ld` elements apart (0: dense).
int check_rows(const phx_kv4_cache *c, phx_dtype t, uint64_t ptr, int64_t heads, int64_t *ld,
               const char *who, const char *what) {
    const int64_t dense = heads * c->head_dim;
    if (!*ld) *ld = dense;
    if (*ld < dense || *ld > kMost || *ld * size_of(t) % 16)
        return set_error(PHX_E_INVALID, "%s: rows of %s must be at least %lld elements apart, in "
                         "whole 16-byte chunks (got %lld)", who, what, (long long)dense,
                         (long long)*ld);
    if (!ptr || (ptr & 15))
        return set_error(PHX_E_INVALID, "%s: %s must be 16-byte aligned", who, what);
    return PHX_OK;
}

PhxKv4 record(const phx_kv4_cache *c, const phx_kv4_batch *b) {
    PhxKv4 p = {};
    p.pool = c->pool;
    p.table = b->table;
    p.lens = b->lens;
    p.q_starts = b->q_starts;
    p.pages = c->pages;
    p.table_stride = b->table_stride;
    p.batch = b->batch;
    p.max_q = b->max_q;
    p.max_len = b->max_len;
    p.rows = b->rows;
    p.heads = c->heads;
    p.page_tokens = c->page_tokens;
    p.splits = 1;
    return p;
}

const char *entry_of(const char *const names[4], phx_dtype t, int head_dim) {
    return names[(t == PHX_F16 ? 0 : 2) + (head_dim == 64 ? 0 : 1)];
}

// append and read: D/8 lanes per unit (the K or V of one row and head)
int move_rows(phx_stream s, const phx_kv4_cache *c, const phx_kv4_batch *b, phx_dtype t,
              uint64_t k, uint64_t v, int64_t ldk, int64_t ldv, const char *who,
              const char *const names[4]) {
    if (!known(t)) return set_error(PHX_E_INVALID, "%s: unknown type %d", who, (int)t);
    if (int rc = check_cache(c, who)) return rc;
    if (int rc = check_batch(b, who)) return rc;
    const bool work = has_work(b);
    if (work)
        if (int rc = check_rows(c, t, k, c->heads, &ldk, who, "K")) return rc;
    if (work)
        if (int rc = check_rows(c, t, v, c->heads, &ldv, who, "V")) return rc;
    const int64_t units = b->batch * 2 * c->heads * b->max_q, per = 256 / (c->head_dim / 8);
    const int64_t groups = (units + per - 1) / per;
    if (work && groups > kMostThreads / 256)
        return set_error(PHX_E_INVALID, "%s: %lld sequences of up to %lld rows are too many", who,
                         (long long)b->batch, (long long)b->max_q);
    if (int rc = on_device((hipStream_t)s)) return rc;
    if (!work) return PHX_OK;
    PhxKv4 p = record(c, b);
    p.x = k;
    p.y = v;
    p.ldx = ldk;
    p.ldy = ldv;
    return launch(kKv4File, entry_of(names, t, c->head_dim), dim3((uint32_t)groups), 256,
                  (hipStream_t)s, &p);
}

}  // namespace

extern "C" {

// ------------------------------------------------------------------ 4-bit weights
size_t phx_w4_packed_bytes(int64_t N, int64_t K) {
    if (N < 0 || K < 0 || !extent(N) || !extent(K)) return 0;
    return (size_t)((N + PHX_W4_TILE_N - 1) / PHX_W4_TILE_N) *
           (size_t)((K + PHX_W4_TILE_K - 1) / PHX_W4_TILE_K) * 1024;
}

int phx_w4_pack(phx_stream s, uint64_t codes, uint64_t packed, int64_t N, int64_t K) {
    if (!extent(N) || !extent(K))
        return set_error(PHX_E_INVALID, "w4_pack: N=%lld K=%lld", (long long)N, (long long)K);
    int64_t words = (int64_t)(phx_w4_packed_bytes(N, K) / 4);
    if (words && (!codes || !packed || (packed & 15)))
        return set_error(PHX_E_INVALID, "w4_pack: null codes, or packed null or not 16-byte aligned");
    if (int rc = on_device((hipStream_t)s)) return rc;
    if (!words) return PHX_OK;
    hipFunction_t f;
    if (int rc = aux_function(kW4File, "w4_pack", &f)) return rc;
    void *args[] = {&codes, &packed, &N, &K, &words};
    const uint32_t grid = (uint32_t)std::min<int64_t>((words + 255) / 256, 1 << 20);
    hipError_t e = hipModuleLaunchKernel(f, grid, 1, 1, 256, 1, 1, 0, (hipStream_t)s, args, nullptr);
    return e == hipSuccess ? PHX_OK : hip_error(e, "w4_pack");
}

int phx_gemv_w4(phx_stream s, phx_dtype t, uint64_t a, uint64_t w, uint64_t scales,
                uint64_t zeros, uint64_t c, int64_t M, int64_t N, int64_t K, int64_t group,
                float alpha, float beta, int64_t lda, int64_t ldc) {
    if (!known(t)) return set_error(PHX_E_INVALID, "gemv_w4: unknown type %d", (int)t);
    if (M < 0 || M > PHX_W4_MAX_ROWS || N < 1 || !extent(N) || K < 8 || K % 8 || !extent(K))
        return set_error(PHX_E_INVALID,
                         "gemv_w4 needs 0 <= M <= %d, N > 0 and K > 0 with K%%8==0 (got %lld,%lld,%lld)",
                         PHX_W4_MAX_ROWS, (long long)M, (long long)N, (long long)K);
    if (N >> 25)  // up to 1024 threads for 16 columns: a launch's 2^32 along an axis
        return set_error(PHX_E_INVALID, "gemv_w4: %lld columns are too many", (long long)N);
    if (group != 32 && group != 64 && group != 128)
        return set_error(PHX_E_INVALID, "gemv_w4: groups of 32, 64 or 128 (got %lld)",
                         (long long)group);
    if (!lda) lda = K;
    if (!ldc) ldc = N;
    const int64_t e = size_of(t);
    if (lda < K || ldc < N || lda > kMost || ldc > kMost || lda * e % 16)
        return set_error(PHX_E_INVALID,
                         "gemv_w4: rows of A must be at least K apart, in whole 16-byte chunks, and "
                         "rows of C at least N (got %lld, %lld)", (long long)lda, (long long)ldc);
    // A is read through a resource of 32-bit offsets
    if (lda * e * PHX_W4_MAX_ROWS > INT32_MAX)
        return set_error(PHX_E_INVALID, "gemv_w4: rows of A too far apart (%lld)", (long long)lda);
    if (M && (!a || !w || !scales || !c)) return set_error(PHX_E_INVALID, "gemv_w4: null operand");
    if (((a | w) & 15) || (scales & 1) || (c & (e - 1)))
        return set_error(PHX_E_INVALID,
                         "gemv_w4: A and the codes must be 16-byte aligned, scales and C by element");
    if (int rc = on_device((hipStream_t)s)) return rc;
    if (M == 0) return PHX_OK;
    PhxGemvW4 p = {a,   w,   scales, zeros, c,    M, N, K, lda, ldc, (K + group - 1) / group,
                   alpha, beta, 0, 1};
    int64_t splits = 1;
    size_t room = 0;
    if (int rc = phx_stream_get_workspace(s, &p.ws, &room)) return rc;
    const W4Form &f = w4_form(t, M, N, K, (int64_t)(room / sizeof(float)) / (M * N), &splits);
    p.splits = (int32_t)splits;
    std::unique_lock<std::mutex> together(split_mutex((hipStream_t)s), std::defer_lock);
    if (splits > 1) together.lock();
    if (int rc = launch(kW4File, f.entry[group == 128 ? 0 : group == 64 ? 1 : 2],
                        dim3((uint32_t)((N + f.columns - 1) / f.columns),
                             (uint32_t)((M + f.rows - 1) / f.rows), (uint32_t)splits),
                        f.threads, (hipStream_t)s, &p))
        return rc;
    if (splits == 1) return PHX_OK;
    return launch(kW4File, t == PHX_F16 ? "gemm_w4_reduce_f16" : "gemm_w4_reduce_f32",
                  dim3((uint32_t)std::min<int64_t>((M * N + 255) / 256, 2048)), 256, (hipStream_t)s,
                  &p);
}

// ------------------------------------------------------------------ 4-bit cache
size_t phx_kv4_page_bytes(int32_t heads, int32_t head_dim, int32_t page_tokens) {
    if (heads < 1 || heads > 1024 || (head_dim != 64 && head_dim != 128)) return 0;
    if (page_tokens != 32 && page_tokens != 64 && page_tokens != 128 && page_tokens != 256) return 0;
    return (size_t)heads * (size_t)page_tokens * (size_t)(head_dim + 8);
}

int phx_kv4_append(phx_stream s, const phx_kv4_cache *cache, const phx_kv4_batch *batch,
                   phx_dtype t, uint64_t k, uint64_t v, int64_t ldk, int64_t ldv) {
    static const char *const names[4] = {"kv4_append_f16_d64", "kv4_append_f16_d128",
                                         "kv4_append_f32_d64", "kv4_append_f32_d128"};
    return move_rows(s, cache, batch, t, k, v, ldk, ldv, "kv4_append", names);
}

int phx_kv4_read(phx_stream s, const phx_kv4_cache *cache, const phx_kv4_batch *batch,
                 phx_dtype t, uint64_t k, uint64_t v, int64_t ldk, int64_t ldv) {
    static const char *const names[4] = {"kv4_read_f16_d64", "kv4_read_f16_d128",
                                         "kv4_read_f32_d64", "kv4_read_f32_d128"};
    return move_rows(s, cache, batch, t, k, v, ldk, ldv, "kv4_read", names);
}

// How an attention runs.  A workgroup takes 4, 8, 16 or 32 columns, a column
// being a row and query head of one KV head: the fewest that hold them all
// (kv4_attend.hip).  Up to 16 columns a workgroup has 8 to 16 waves instead of
// four where there are fewer than kAttendFull like it and kAttendWide keys or
// more to share out, half of them in a part of a split (32 sequences, 8 x 4 heads
// of 128: 512 keys 9.4 us with 4 waves, 10.0 with 12; 2048 keys 23.7 and 19.3; one
// sequence of 4096 in 16 parts 9.9 and 11.1).  Above 64 columns it takes 128
// of them, with no wave of its own for a share of the keys, where that gives
// kAttendChunks workgroups (16 KV heads of 128 x 1000 columns over 4133 keys:
// 211 us against 353; 64 x 256 columns over 4000: 113 against 104; 24 x 800 over
// 1000: 49 against 53).  The keys are split further (those of the longest
// sequence there can be) to bring the launch to kAttendGroups workgroups, into
// parts of at least kAttendPart keys and at most PHX_KV4_SPLITS of them, where that
// spares a workgroup kAttendSaved keys, and one more for 32 rows' and heads' parts,
// as joining the parts is a launch more (one sequence, 8 x 4 heads of 128: 4096
// keys in parts of 256 9.9 us, of 512 12.4, of 1024 14.3; 512 keys whole 8.1, in two
// 9.9; 24 sequences of 1024, 4 heads, f32: whole 11.2, in two 12.8; 2 x 300 rows over
// 1200 keys, 2 x 2 heads: whole 28.3, in three 35.5).
static const int64_t kAttendFull = 512, kAttendWide = 1024, kAttendChunks = 160,
                     kAttendGroups = 256, kAttendPart = 256, kAttendSaved = 768;
struct AttendForm {
    int64_t columns;
    uint32_t waves;  // of the wide form
    const char *entry[2][4];
};
#define ENTRIES(tail)                                                          \
    {"kv4_attend_f16_d64_" tail, "kv4_attend_f16_d128_" tail,                  \
     "kv4_attend_f32_d64_" tail, "kv4_attend_f32_d128_" tail}
static const AttendForm kAttendForms[] = {
    {4, 12, {ENTRIES("c1_g4_w4"), ENTRIES("c1_g4_w12")}},
    {8, 16, {ENTRIES("c1_g2_w4"), ENTRIES("c1_g2_w16")}},
    {16, 8, {ENTRIES("c1_g1_w4"), ENTRIES("c1_g1_w8")}},
    {32, 4, {ENTRIES("c2_g1_w4"), ENTRIES("c2_g1_w4")}},
    {128, 4, {ENTRIES("chunk"), ENTRIES("chunk")}}};
#undef ENTRIES

static int64_t attend_groups(const phx_kv4_batch *b, int64_t ratio, const AttendForm &f) {
    return (b->max_q * ratio + f.columns - 1) / f.columns;
}

static const AttendForm &attend_form(const phx_kv4_cache *c, const phx_kv4_batch *b,
                                     int64_t ratio) {
    const int64_t columns = b->max_q * ratio;
    const AttendForm &chunk = kAttendForms[4];
    if (columns > 64 && b->batch * c->heads * attend_groups(b, ratio, chunk) >= kAttendChunks)
        return chunk;
    int i = 0;
    while (i < 3 && kAttendForms[i].columns < columns) ++i;
    return kAttendForms[i];
}

static size_t split_bytes(const phx_kv4_cache *c, const phx_kv4_batch *b, int64_t q_heads) {
    return (size_t)b->rows * (size_t)q_heads * (size_t)(c->head_dim + 2) * sizeof(float);
}

// The most keys that a sequence can have.
static int64_t longest(const phx_kv4_cache *c, const phx_kv4_batch *b) {
    return std::min(b->max_len, b->table_stride * c->page_tokens);
}

static int64_t attend_splits(const phx_kv4_cache *c, const phx_kv4_batch *b, int64_t q_heads) {
    const int64_t ratio = q_heads / c->heads;
    const int64_t groups = b->batch * c->heads *
                           attend_groups(b, ratio, attend_form(c, b, ratio));
    const int64_t keys = longest(c, b);
    if (!has_work(b)) return 1;
    const int64_t splits = std::max<int64_t>(
        1, std::min({kAttendGroups / groups, keys / kAttendPart, (int64_t)PHX_KV4_SPLITS}));
    if (splits == 1) return 1;  // (else there are few rows)
    const int64_t parts = b->batch * b->max_q * q_heads * splits;
    return keys - keys / splits < kAttendSaved + parts / 32 ? 1 : splits;
}

static int check_heads(const phx_kv4_cache *c, int64_t q_heads, const char *who) {
    if (q_heads < 1 || q_heads % c->heads || q_heads > 65535)
        return set_error(PHX_E_INVALID, "%s: %lld query heads over %d KV heads", who,
                         (long long)q_heads, c->heads);
    return PHX_OK;
}

int phx_kv4_split_plan(const phx_kv4_cache *cache, const phx_kv4_batch *batch, int64_t q_heads,
                       int *splits, size_t *workspace_bytes) {
    if (int rc = check_cache(cache, "kv4_split_plan")) return rc;
    if (int rc = check_batch(batch, "kv4_split_plan")) return rc;
    if (int rc = check_heads(cache, q_heads, "kv4_split_plan")) return rc;
    const int64_t sp = attend_splits(cache, batch, q_heads);
    if (splits) *splits = (int)sp;
    if (workspace_bytes) *workspace_bytes = sp > 1 ? (size_t)sp * split_bytes(cache, batch, q_heads) : 0;
    return PHX_OK;
}

int phx_kv4_attention(phx_stream s, const phx_kv4_cache *cache, const phx_kv4_batch *batch,
                      phx_dtype t, uint64_t q, uint64_t o, int64_t q_heads, float scale,
                      int causal, int64_t ldq, int64_t ldo) {
    static const char *const combine[4] = {"kv4_combine_f16_d64", "kv4_combine_f16_d128",
                                           "kv4_combine_f32_d64", "kv4_combine_f32_d128"};
    const char *who = "kv4_attention";
    if (!known(t)) return set_error(PHX_E_INVALID, "%s: unknown type %d", who, (int)t);
    if (int rc = check_cache(cache, who)) return rc;
    if (int rc = check_batch(batch, who)) return rc;
    if (int rc = check_heads(cache, q_heads, who)) return rc;
    const bool work = has_work(batch);
    if (work)
        if (int rc = check_rows(cache, t, q, q_heads, &ldq, who, "Q")) return rc;
    if (work)
        if (int rc = check_rows(cache, t, o, q_heads, &ldo, who, "O")) return rc;
    const int64_t ratio = q_heads / cache->heads;
    const AttendForm &form = attend_form(cache, batch, ratio);
    const int64_t each = attend_groups(batch, ratio, form);
    const int64_t groups = batch->batch * cache->heads * each;
    const int64_t units = batch->batch * batch->max_q * q_heads;
    // (the workgroups of a form, and of the one that joins the parts of a split)
    const int64_t planned = attend_splits(cache, batch, q_heads);
    if (work && (groups > kMostThreads / 1024 / planned || (planned > 1 && units > kMostThreads / 512)))
        return set_error(PHX_E_INVALID, "%s: %lld sequences of up to %lld rows are too many", who,
                         (long long)batch->batch, (long long)batch->max_q);
    if (int rc = on_device((hipStream_t)s)) return rc;
    if (!work) return PHX_OK;
    PhxKv4 p = record(cache, batch);
    p.x = q;
    p.y = o;
    p.ldx = ldq;
    p.ldy = ldo;
    p.ratio = (int32_t)ratio;
    p.causal = causal != 0;
    p.scale = scale;
    p.groups = (int32_t)each;
    size_t room = 0;
    if (int rc = phx_stream_get_workspace(s, &p.ws, &room)) return rc;
    const size_t part = split_bytes(cache, batch, q_heads);
    p.splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>(planned, (int64_t)(room / part)));
    const bool wide = form.columns <= 16 && groups < kAttendFull &&
                      longest(cache, batch) / p.splits >=
                          (p.splits > 1 ? kAttendWide / 2 : kAttendWide);
    std::unique_lock<std::mutex> together(split_mutex((hipStream_t)s), std::defer_lock);
    if (p.splits > 1) together.lock();
    if (int rc = launch(kAttendFile, entry_of(form.entry[wide], t, cache->head_dim),
                        dim3((uint32_t)(each * p.splits), (uint32_t)cache->heads,
                             (uint32_t)batch->batch),
                        64 * (wide ? form.waves : 4), (hipStream_t)s, &p))
        return rc;
    if (p.splits == 1) return PHX_OK;
    return launch(kAttendFile, entry_of(combine, t, cache->head_dim),
                  dim3((uint32_t)units), 512, (hipStream_t)s, &p);
}

// ------------------------------------------------------------------ pages
int phx_pages_copy(phx_stream s, uint64_t pool, int64_t pages, size_t page_bytes,
                   const int32_t *src, const int32_t *dst, int64_t n, int64_t layers,
                   uint64_t layer_stride) {
    if (pages < 1 || !extent(pages) || !page_bytes || page_bytes % 16 || page_bytes > (1u << 30))
        return set_error(PHX_E_INVALID, "pages_copy: %lld pages of %zu bytes", (long long)pages,
                         page_bytes);
    if (layers < 0 || layers > 65535 || (layers > 1 && (layer_stride % 16 ||
                                                         layer_stride / (uint64_t)pages < page_bytes)))
        return set_error(PHX_E_INVALID, "pages_copy: %lld layers %llu bytes apart", (long long)layers,
                         (unsigned long long)layer_stride);
    if (n < 0 || (n > 0 && (!src || !dst)))
        return set_error(PHX_E_INVALID, "pages_copy: null list");
    if (n && layers && (!pool || (pool & 15)))
        return set_error(PHX_E_INVALID, "pages_copy: the pool must be 16-byte aligned");
    // (one layer is below 2^61 bytes)
    const uint64_t last = layers ? UINT64_MAX - (uint64_t)pages * page_bytes : 0;
    if (n && layers && (pool > last || (layers > 1 && layer_stride > (last - pool) / (uint64_t)(layers - 1))))
        return set_error(PHX_E_INVALID, "pages_copy: %lld layers %llu bytes apart end past the address space",
                         (long long)layers, (unsigned long long)layer_stride);
    try {
        std::vector<int32_t> from, to;
        from.reserve((size_t)n);
        to.reserve((size_t)n);
        for (int64_t i = 0; i < n; ++i) {
            if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages)
                return set_error(PHX_E_INVALID, "pages_copy: copy %lld, %d to %d, of %lld pages",
                                 (long long)i, src[i], dst[i], (long long)pages);
            if (src[i] == dst[i]) continue;
            from.push_back(src[i]);
            to.push_back(dst[i]);
        }
        std::vector<int32_t> a(from), b(to);
        std::sort(a.begin(), a.end());
        std::sort(b.begin(), b.end());
        for (size_t i = 0; i < b.size(); ++i)
            if ((i && b[i] == b[i - 1]) || std::binary_search(a.begin(), a.end(), b[i]))
                return set_error(PHX_E_INVALID,
                                 "pages_copy: page %d is the destination of several copies, or "
                                 "destination and source", b[i]);
        if (int rc = on_device((hipStream_t)s)) return rc;
        if (!layers) return PHX_OK;
        PhxPagesCopy p;
        p.pool = pool;
        p.page_bytes = page_bytes;
        p.layer_stride = layer_stride;
        const uint32_t groups = (uint32_t)((page_bytes / 16 + 4 * PHX_PAGES_THREADS - 1) /
                                           (4 * PHX_PAGES_THREADS));
        for (size_t at = 0; at < from.size(); at += PHX_PAGES_PER_LAUNCH) {
            const size_t m = std::min<size_t>(from.size() - at, PHX_PAGES_PER_LAUNCH);
            std::copy_n(from.begin() + at, m, p.src);
            std::copy_n(to.begin() + at, m, p.dst);
            if (int rc = launch(kPagesFile, "pages_copy", dim3(groups, (uint32_t)m, (uint32_t)layers),
                                PHX_PAGES_THREADS, (hipStream_t)s, &p))
                return rc;
        }
    } catch (const std::exception &e) {
        return set_error(PHX_E_EXHAUSTED, "pages_copy: %s", e.what());
    }
    return PHX_OK;
}

}  // extern "C"
