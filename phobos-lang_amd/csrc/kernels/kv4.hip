// Attention over keys and values held in 4 bits in pages, and the writes and
// reads of those pages (the layout and the arithmetic: include/phobos_hip.h,
// phx_kv4_*).
#include "phx_common.h"
#include "phx_decode.h"

namespace {

// A sequence of the call: its tokens, and its rows' first index and count.
struct Seq {
    int64_t tokens, row0, count;
};

__device__ __forceinline__ Seq kv4_seq(const PhxKv4 &p, int64_t b) {
    Seq s;
    int64_t most = p.table_stride * p.page_tokens;
    if (p.max_len < most) most = p.max_len;
    s.tokens = ((const int32_t *)p.lens)[b];
    s.tokens = s.tokens < 0 ? 0 : s.tokens > most ? most : s.tokens;
    s.row0 = b * p.max_q;
    s.count = p.max_q;
    if (p.q_starts) {
        const int32_t *q = (const int32_t *)p.q_starts + b;
        s.row0 = q[0];
        const int64_t n = (int64_t)q[1] - q[0];
        s.count = n < 0 ? 0 : n > p.max_q ? p.max_q : n;
    }
    return s;
}

// The page of a sequence's token, or -1.
__device__ __forceinline__ int64_t kv4_page(const PhxKv4 &p, int64_t b, int64_t token) {
    const int64_t page = ((const int32_t *)p.table)[b * p.table_stride + token / p.page_tokens];
    return page >= 0 && page < p.pages ? page : -1;
}

// A page's bytes of one head.
template <int D>
__device__ __forceinline__ char *kv4_head(const PhxKv4 &p, int64_t page, int head) {
    return (char *)p.pool + (page * p.heads + head) * ((int64_t)p.page_tokens * (D + 8));
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
__device__ __forceinline__ void load8(const T *src, float *x) {
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
    const T *src = u.v ? (const T *)p.y + u.row * p.ldy : (const T *)p.x + u.row * p.ldx;
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
    char *head = kv4_head<D>(p, page, u.head);
    const uint32_t slot = (uint32_t)(u.token % p.page_tokens);
    *(uint32_t *)(head + kv4_word<D>(p.page_tokens, u.v, slot, e)) = word;
    if (e == 0) {
        phx_h2 pair;
        pair.x = sc;
        pair.y = m;
        *(phx_h2 *)(head + kv4_param<D>(p.page_tokens, u.v, slot)) = pair;
    }
}

template <typename T, int D>
__device__ __forceinline__ void read(const PhxKv4 &p) {
    constexpr int L = D / 8;
    const int e = threadIdx.x % L;
    const Unit u = kv4_unit<D>(p, (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L);
    if (!u.live) return;
    T *dst = (u.v ? (T *)p.y + u.row * p.ldy : (T *)p.x + u.row * p.ldx) + u.head * D + e * 8;
    const int64_t page = u.token < 0 ? -1 : kv4_page(p, u.b, u.token);
    float x[8] = {};
    if (page >= 0) {
        const char *head = kv4_head<D>(p, page, u.head);
        const uint32_t slot = (uint32_t)(u.token % p.page_tokens);
        const uint32_t word = *(const uint32_t *)(head + kv4_word<D>(p.page_tokens, u.v, slot, e));
        const phx_h2 pair = *(const phx_h2 *)(head + kv4_param<D>(p.page_tokens, u.v, slot));
        for (int i = 0; i < 8; ++i)
            x[i] = (float)((word >> (4 * i)) & 15) * (float)pair.x + (float)pair.y;
    }
    for (int i = 0; i < 8; ++i) dst[i] = (T)x[i];
}

// One wave per row and query head; 64 keys at a time, a key per lane for the
// scores, D/64 elements per lane for the sums.
template <typename T, int D>
__device__ __forceinline__ void attend(const PhxKv4 &p) {
    __shared__ float qs[D], ps[64], vs[64];
    const int lane = threadIdx.x;
    const int64_t b = blockIdx.z, i = blockIdx.x;
    const int qh = blockIdx.y, head = qh / p.ratio;
    const Seq s = kv4_seq(p, b);
    const int64_t row = s.row0 + i;
    if (i >= s.count || row < 0 || row >= p.rows) return;
    int64_t keys = s.tokens;
    if (p.causal) keys = s.tokens - s.count + i + 1;
    const T *q = (const T *)p.x + row * p.ldx + qh * D;
    for (int d = lane; d < D; d += 64) qs[d] = (float)q[d];
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[D / 64] = {};
    for (int64_t k0 = 0; k0 < keys; k0 += 64) {
        const int64_t t = k0 + lane;
        float sc = -INFINITY;
        const int64_t page = t < keys ? kv4_page(p, b, t) : -1;
        if (page >= 0) {
            const char *h = kv4_head<D>(p, page, head);
            const uint32_t slot = (uint32_t)(t % p.page_tokens);
            const phx_h2 kp = *(const phx_h2 *)(h + kv4_param<D>(p.page_tokens, false, slot));
            float dot = 0.0f;
            for (int e = 0; e < D / 8; ++e) {
                const uint32_t w = *(const uint32_t *)(h + kv4_word<D>(p.page_tokens, false, slot, e));
                for (int u = 0; u < 8; ++u)
                    dot = fmaf(qs[e * 8 + u],
                               (float)((w >> (4 * u)) & 15) * (float)kp.x + (float)kp.y, dot);
            }
            sc = dot * p.scale;
        }
        float top = sc;
        for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        if (top == -INFINITY) continue;
        const float mn = fmaxf(m, top), f = expf(m - mn);
        const float pr = expf(sc - mn);
        float sum = pr;
        for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
        l = l * f + sum;
        m = mn;
        ps[lane] = pr;
        __syncthreads();
        for (int x = 0; x < D / 64; ++x) o[x] *= f;
        for (int u = 0; u < 64; ++u) {
            const int64_t tu = k0 + u;
            const int64_t pg = tu < keys ? kv4_page(p, b, tu) : -1;
            if (pg < 0) continue;
            const char *h = kv4_head<D>(p, pg, head);
            const uint32_t slot = (uint32_t)(tu % p.page_tokens);
            const phx_h2 vp = *(const phx_h2 *)(h + kv4_param<D>(p.page_tokens, true, slot));
            for (int x = 0; x < D / 64; ++x) {
                const int d = lane + 64 * x;
                const uint32_t w =
                    *(const uint32_t *)(h + kv4_word<D>(p.page_tokens, true, slot, d / 8));
                const float v = (float)((w >> (4 * (d % 8))) & 15) * (float)vp.x + (float)vp.y;
                o[x] = fmaf(ps[u], v, o[x]);
            }
        }
        __syncthreads();
    }
    T *out = (T *)p.y + row * p.ldy + qh * D;
    for (int x = 0; x < D / 64; ++x) out[lane + 64 * x] = (T)(l > 0.0f ? o[x] / l : l);
}

}  // namespace

#define KV4(T, D, suffix)                                                                       \
    extern "C" __global__ __launch_bounds__(256) void kv4_append_##suffix(PhxKv4 p) {           \
        append<T, D>(p);                                                                        \
    }                                                                                           \
    extern "C" __global__ __launch_bounds__(256) void kv4_read_##suffix(PhxKv4 p) {             \
        read<T, D>(p);                                                                          \
    }                                                                                           \
    extern "C" __global__ __launch_bounds__(64) void kv4_attend_##suffix(PhxKv4 p) {            \
        attend<T, D>(p);                                                                        \
    }
KV4(_Float16, 64, f16_d64)
KV4(_Float16, 128, f16_d128)
KV4(float, 64, f32_d64)
KV4(float, 128, f32_d128)
