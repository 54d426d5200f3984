// Writes and reads of pages that hold keys and values in 4 bits (the layout and
// the arithmetic: include/phobos_hip.h, phx_kv4_append and phx_kv4_read).
//
// One pass, bound by the rows' bytes and, with few rows, by the launch: D/8 lanes
// take the K or V of a row and head, 16-byte chunks next to each other, and find
// the row's range among themselves. 2 x 2000 rows of 8 heads of 128, f32: 9.5 us
// written (3.9 TB/s), 8.5 us read back (4.4 TB/s); 32 f16 rows 3.1 and 2.5 us.
#include "kv4.h"

namespace {

struct Unit {  // D/8 lanes: the K or V of one row and head
    int64_t row, token;  // token: its position; may be below 0
    uint32_t b, head;
    bool v, live;
};

// Lanes go over the units with the rows of a head fastest, so that a wave's V
// dwords of neighbouring tokens are neighbours too.  (Units are below 2^31.)
template <int D>
__device__ __forceinline__ Unit kv4_unit(const PhxKv4 &p) {
    constexpr uint32_t L = D / 8;
    Unit r;
    uint32_t u = blockIdx.x * (256 / L) + threadIdx.x / L;
    const uint32_t max_q = (uint32_t)p.max_q, i = u % max_q;
    u /= max_q;
    r.head = u % p.heads;
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

// A unit's token's part of a page, or null.
template <int D>
__device__ __forceinline__ PHX_GLOBAL char *kv4_part(const PhxKv4 &p, const Unit &u, uint32_t *slot) {
    if (u.token < 0) return nullptr;
    const uint32_t P = p.page_tokens, token = (uint32_t)u.token;
    *slot = token & (P - 1);
    const int32_t page = ((const PHX_GLOBAL int32_t *)p.table)[u.b * p.table_stride +
                                                               (token >> __builtin_ctz(P))];
    return page >= 0 && page < p.pages ? kv4_head<D>(p, page, u.head) : nullptr;
}

// A lane's eight elements of its unit, in chunks of 16 bytes that are next to its
// neighbours': f16 8 e .. 8 e + 7; f32 4 e .. and 4 (e + D/8) .., halves of the
// octets e / 2 and e / 2 + D/16 (32 bytes a lane, in two accesses that leave
// every other 16 out: reading back 32.8 MB 10.8 us, with these 8.5).
template <typename T, int D>
__device__ __forceinline__ void load8(const PHX_GLOBAL T *src, uint32_t e, float *x) {
    if constexpr (sizeof(T) == 2) {
        const phx_h8 w = *(const PHX_GLOBAL phx_h8 *)(src + 8 * e);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)w[i];
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const phx_f4 w = *(const PHX_GLOBAL phx_f4 *)(src + 4 * (e + h * (D / 8)));
#pragma unroll
            for (int i = 0; i < 4; ++i) x[4 * h + i] = w[i];
        }
    }
}
template <typename T, int D>
__device__ __forceinline__ void store8(PHX_GLOBAL T *dst, uint32_t e, const float *x) {
    if constexpr (sizeof(T) == 2) {
        phx_h8 w;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = (_Float16)x[i];
        *(PHX_GLOBAL phx_h8 *)(dst + 8 * e) = w;
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const phx_f4 w = {x[4 * h], x[4 * h + 1], x[4 * h + 2], x[4 * h + 3]};
            *(PHX_GLOBAL phx_f4 *)(dst + 4 * (e + h * (D / 8))) = w;
        }
    }
}

// f16(f32((hi - lo) / 15)), the quotient in 64 bits: f32's is 2^-22 of it off at
// most, and settles it where that moves no rounding.
__device__ __forceinline__ _Float16 step_of(float lo, float hi) {
    const float y = (hi - lo) * (1.0f / 15.0f);
    const _Float16 a = (_Float16)(y * (1.0f - 0x1p-21f)), b = (_Float16)(y * (1.0f + 0x1p-21f));
    return a == b ? a : (_Float16)(float)(((double)hi - (double)lo) / 15.0);
}

// rint((x - m) / s) in 0 .. 15, of the exact quotient, 0 for none.
__device__ __forceinline__ uint32_t code_of(float x, float m, float s, float inverse) {
    // the difference, the inverse (1 ulp) and the product: 2^-22 of a quotient off
    // at most, so 2^-18 where it counts; a quotient that near a tie is taken
    // again in 64 bits, one in 2^15 of ordinary ones (a 64-bit division for all
    // takes longer than the memory does: 32.8 MB of f32 14.4 us, with this 9.5)
    const float q = (x - m) * inverse;
    float c = rintf(q);
    if (fabsf(q - c) > 0.5f - 0x1p-16f && q > 0.0f && q < 16.0f)
        c = (float)rint(((double)x - (double)m) / (double)s);
    return (uint32_t)fminf(fmaxf(c, 0.0f), 15.0f);
}

template <typename T, int D>
__device__ __forceinline__ void append(const PhxKv4 &p) {
    constexpr int L = D / 8;
    const uint32_t e = threadIdx.x % L;
    const Unit u = kv4_unit<D>(p);
    if (!u.live) return;
    float x[8];
    load8<T, D>((u.v ? (const PHX_GLOBAL T *)p.y + u.row * p.ldy
                     : (const PHX_GLOBAL T *)p.x + u.row * p.ldx) + u.head * D, e, x);
    uint32_t slot;
    PHX_GLOBAL char *head = kv4_part<D>(p, u, &slot);
    if (!head) return;
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
#pragma unroll
    for (int s = 1; s < L; s <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, s));
        hi = fmaxf(hi, __shfl_xor(hi, s));
    }
    phx_h2 pair = {step_of(lo, hi), (_Float16)lo};
    if (pair.x < (_Float16)0x1p-24f) pair.x = (_Float16)0x1p-24f;
    const float s = (float)pair.x, m = (float)pair.y, inverse = __builtin_amdgcn_rcpf(s);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) word |= code_of(x[i], m, s, inverse) << (4 * i);
    uint32_t octet = e;
    if (sizeof(T) == 4) {
        // of two lanes with halves of two octets, each puts one together
        const bool odd = e & 1;
        const uint32_t other = __builtin_amdgcn_mov_dpp(odd ? word & 0xffff : word >> 16,
                                                        0xb1, 0xf, 0xf, true);
        word = odd ? other | (word & 0xffff0000u) : (word & 0xffff) | other << 16;
        octet = e / 2 + (odd ? L / 2 : 0);
    }
    *(PHX_GLOBAL uint32_t *)(head + kv4_word<D>(p.page_tokens, u.v, slot, octet)) = word;
    if (e == 0)
        *(PHX_GLOBAL uint32_t *)(head + kv4_param<D>(p.page_tokens, u.v, slot)) =
            __builtin_bit_cast(uint32_t, pair);
}

template <typename T, int D>
__device__ __forceinline__ void read(const PhxKv4 &p) {
    constexpr int L = D / 8;
    const uint32_t e = threadIdx.x % L;
    const Unit u = kv4_unit<D>(p);
    if (!u.live) return;
    uint32_t slot;
    const PHX_GLOBAL char *head = kv4_part<D>(p, u, &slot);
    float x[8] = {};
    if (head) {
        auto octet = [&](uint32_t o) {
            return *(const PHX_GLOBAL uint32_t *)(head + kv4_word<D>(p.page_tokens, u.v, slot, o));
        };
        uint32_t word;
        if constexpr (sizeof(T) == 2) {
            word = octet(e);
        } else {
            const uint32_t half = e % 2 * 16;
            word = (octet(e / 2) >> half & 0xffff) | octet(e / 2 + L / 2) >> half << 16;
        }
        const phx_h2 pair =
            *(const PHX_GLOBAL phx_h2 *)(head + kv4_param<D>(p.page_tokens, u.v, slot));
        const float s = (float)pair.x, m = (float)pair.y;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)((word >> (4 * i)) & 15) * s + m;
    }
    store8<T, D>((u.v ? (PHX_GLOBAL T *)p.y + u.row * p.ldy
                      : (PHX_GLOBAL T *)p.x + u.row * p.ldx) + u.head * D, e, x);
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
