// Writes and reads of pages that hold keys and values in 4 bits (the layout and
// the arithmetic: include/phobos_hip.h, phx_kv4_append and phx_kv4_read).
#include "kv4.h"

namespace {

struct Unit {  // D/8 lanes: the K or V of one row and head
    int64_t b, row;
    int head;
    bool v, live;
    int64_t token;  // its position; may be below 0
};

// Lanes go over the units with the rows of a head fastest, so that a wave's V
// dwords of neighbouring tokens are neighbours too.
template <int D>
__device__ __forceinline__ Unit kv4_unit(const PhxKv4 &p, int64_t u) {
    Unit r;
    const int64_t i = u % p.max_q;
    u /= p.max_q;
    r.head = (int)(u % p.heads);
    u /= p.heads;
    r.v = u & 1;
    r.b = u >> 1;
    r.live = r.b < p.batch;
    if (!r.live) return r;
    const Seq s = kv4_seq(p, r.b);
    r.row = s.row0 + i;
    r.live = i < s.count && r.row >= 0 && r.row < p.rows;
    r.token = s.tokens - s.count + i;
    return r;
}

template <typename T>
__device__ __forceinline__ void load8(const PHX_GLOBAL T *src, float *x) {
    for (int i = 0; i < 8; ++i) x[i] = (float)src[i];
}

template <typename T, int D>
__device__ __forceinline__ void append(const PhxKv4 &p) {
    constexpr int L = D / 8;
    const int e = threadIdx.x % L;
    const Unit u = kv4_unit<D>(p, (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L);
    if (!u.live || u.token < 0) return;
    const int64_t page = kv4_page(p, u.b, u.token);
    if (page < 0) return;
    const PHX_GLOBAL T *src = u.v ? (const PHX_GLOBAL T *)p.y + u.row * p.ldy
                                  : (const PHX_GLOBAL T *)p.x + u.row * p.ldx;
    float x[8];
    load8(src + u.head * D + e * 8, x);
    float lo = x[0], hi = x[0];
    for (int i = 1; i < 8; ++i) lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
    for (int s = 1; s < L; s <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, s));
        hi = fmaxf(hi, __shfl_xor(hi, s));
    }
    // in 64 bits: the quotient's ties are those of the exact values
    const _Float16 m = (_Float16)lo;
    _Float16 sc = (_Float16)(float)(((double)hi - (double)lo) / 15.0);
    if ((float)sc < 0x1p-24f) sc = (_Float16)0x1p-24f;
    uint32_t word = 0;
    for (int i = 0; i < 8; ++i) {
        const double c = rint(((double)x[i] - (double)(float)m) / (double)(float)sc);
        word |= (c > 0.0 ? c < 15.0 ? (uint32_t)c : 15u : 0u) << (4 * i);
    }
    PHX_GLOBAL char *head = kv4_head<D>(p, page, u.head);
    const uint32_t slot = (uint32_t)(u.token % p.page_tokens);
    *(PHX_GLOBAL uint32_t *)(head + kv4_word<D>(p.page_tokens, u.v, slot, e)) = word;
    if (e == 0) {
        phx_h2 pair;
        pair.x = sc;
        pair.y = m;
        *(PHX_GLOBAL phx_h2 *)(head + kv4_param<D>(p.page_tokens, u.v, slot)) = pair;
    }
}

template <typename T, int D>
__device__ __forceinline__ void read(const PhxKv4 &p) {
    constexpr int L = D / 8;
    const int e = threadIdx.x % L;
    const Unit u = kv4_unit<D>(p, (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L);
    if (!u.live) return;
    PHX_GLOBAL T *dst = (u.v ? (PHX_GLOBAL T *)p.y + u.row * p.ldy
                             : (PHX_GLOBAL T *)p.x + u.row * p.ldx) + u.head * D + e * 8;
    const int64_t page = u.token < 0 ? -1 : kv4_page(p, u.b, u.token);
    float x[8] = {};
    if (page >= 0) {
        const PHX_GLOBAL char *head = kv4_head<D>(p, page, u.head);
        const uint32_t slot = (uint32_t)(u.token % p.page_tokens);
        const uint32_t word = *(const PHX_GLOBAL uint32_t *)(head + kv4_word<D>(p.page_tokens, u.v, slot, e));
        const phx_h2 pair = *(const PHX_GLOBAL phx_h2 *)(head + kv4_param<D>(p.page_tokens, u.v, slot));
        for (int i = 0; i < 8; ++i)
            x[i] = (float)((word >> (4 * i)) & 15) * (float)pair.x + (float)pair.y;
    }
    for (int i = 0; i < 8; ++i) dst[i] = (T)x[i];
}

}  // namespace

#define KV4(T, D, suffix)                                                                       \
    extern "C" __global__ __launch_bounds__(256) void kv4_append_##suffix(PhxKv4 p) {           \
        append<T, D>(p);                                                                        \
    }                                                                                           \
    extern "C" __global__ __launch_bounds__(256) void kv4_read_##suffix(PhxKv4 p) {             \
        read<T, D>(p);                                                                          \
    }
KV4(_Float16, 64, f16_d64)
KV4(_Float16, 128, f16_d128)
KV4(float, 64, f32_d64)
KV4(float, 128, f32_d128)
