// What the host runtime and the decode kernels (gemv_w4.hip, kv4.hip,
// pages.hip) share: their argument records and launch geometry.
#pragma once
#include <stdint.h>

#define PHX_W4_MAX_ROWS 64
#define PHX_W4_TILE_N 16
#define PHX_W4_TILE_K 128

struct PhxGemvW4 {
    uint64_t a, w, scales, zeros, c;
    int64_t M, N, K, lda, ldc, groups;
    float alpha, beta;
    uint64_t ws;
    int32_t splits;
};

// A kv4 call: the cache, its sequences, and the tensors of their rows.
// Element strides.
struct PhxKv4 {
    uint64_t pool, table, lens, q_starts;
    int64_t pages, table_stride, batch, max_q, max_len, rows;
    int32_t heads, page_tokens;
    uint64_t x, y;  // append, read: K and V; attention: Q and O
    int64_t ldx, ldy;
    uint64_t ws;
    int32_t ratio, splits, causal, groups;  // groups: of columns, per KV head
    float scale;
};

#define PHX_KV4_SPLITS 128  // the most parts of a sequence's keys

// A call's copies of pages, by value: a launch carries its lists itself.
#define PHX_PAGES_PER_LAUNCH 448
struct PhxPagesCopy {
    uint64_t pool, page_bytes, layer_stride;
    int32_t src[PHX_PAGES_PER_LAUNCH], dst[PHX_PAGES_PER_LAUNCH];
};
#define PHX_PAGES_THREADS 256
