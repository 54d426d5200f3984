// The 4-bit cache as the kernels see it: a call's sequences, and where a
// token's codes and parameters lie (include/phobos_hip.h, phx_kv4_*).
#pragma once
#include "phx_common.h"
#include "phx_decode.h"

// Addresses arrive as integers: without their address space they would be
// accessed with flat instructions, which also take the LDS path.
#define PHX_GLOBAL __attribute__((address_space(1)))

namespace {

// A sequence of the call: its tokens, and its rows' first index and count.
struct Seq {
    int64_t tokens, row0, count;
};

__device__ __forceinline__ Seq kv4_seq(const PhxKv4 &p, int64_t b) {
    Seq s;
    int64_t most = p.table_stride * p.page_tokens;
    if (p.max_len < most) most = p.max_len;
    s.tokens = ((const PHX_GLOBAL int32_t *)p.lens)[b];
    s.tokens = s.tokens < 0 ? 0 : s.tokens > most ? most : s.tokens;
    s.row0 = b * p.max_q;
    s.count = p.max_q;
    if (p.q_starts) {
        const PHX_GLOBAL int32_t *q = (const PHX_GLOBAL int32_t *)p.q_starts + b;
        s.row0 = q[0];
        const int64_t n = (int64_t)q[1] - q[0];
        s.count = n < 0 ? 0 : n > p.max_q ? p.max_q : n;
    }
    return s;
}

// A page's bytes of one head.
template <int D>
__device__ __forceinline__ PHX_GLOBAL char *kv4_head(const PhxKv4 &p, int64_t page, int head) {
    return (PHX_GLOBAL char *)p.pool + (page * p.heads + head) * ((int64_t)p.page_tokens * (D + 8));
}

// Byte offset of the dword with elements 8e .. 8e+7 of a token, in a head's
// part of a page.
template <int D>
__device__ __forceinline__ uint32_t kv4_word(uint32_t P, bool v, uint32_t slot, uint32_t e) {
    if (!v) return slot * (D / 2) + e * 4;
    return P * (D / 2) + (((slot / 4) * (D / 8) + e) * 4 + slot % 4) * 4;
}
// Byte offset of a token's (scale, minimum).
template <int D>
__device__ __forceinline__ uint32_t kv4_param(uint32_t P, bool v, uint32_t slot) {
    return P * D + (v ? 4 * P : 0) + 4 * slot;
}

}  // namespace
