// Products of rows and weights in 8 bits, dense and grouped by expert (the layout
// and the arithmetic: include/phobos_hip.h, phx_gemm_f8 and phx_gemm_f8_grouped).
//
//   acc[m,n] = sum over blocks b of sa[m,b] sw[n/128,b] * sum over k in b of a[m,k] w[n,k]
//
// The inner sum is one v_mfma_f32_16x16x128 of the codes, scaled in f32. The
// weights are its A operand, so that a lane holds four neighbouring columns of
// one row of C, and one row's scale.
#include "f8.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void *lds_ptr;
typedef __attribute__((address_space(8))) void *rsrc_ptr;

constexpr uint32_t kNone = 0x80000000u;  // an offset past every resource's end: zeros

// Where a tile of TM rows lies: its expert, and C's rows from m0 up to end.
struct Tile {
    int64_t m0, end, expert;
    uint32_t column;  // in tiles
    bool live;
};

__device__ __forceinline__ int64_t cut(int64_t v, int64_t most) {
    return v < 0 ? 0 : v > most ? most : v;
}

// Tiles of the groups in their order, `columns` of them for every TM rows; the
// groups' ranges are made to ascend, so that none overlap whatever the starts hold.
template <int TM>
__device__ __forceinline__ Tile tile_of(const PhxF8Gemm &p, uint32_t columns) {
    Tile t;
    const uint32_t id = blockIdx.x;
    const int64_t wanted = id / columns;
    t.column = id % columns;
    t.expert = 0;
    t.live = false;
    if (!p.starts) {
        t.m0 = wanted * TM;
        t.end = p.M;
        t.live = t.m0 < p.M;
        return t;
    }
    const uint32_t lane = threadIdx.x & 63;
    int64_t before = 0, floor = 0;  // tiles of the experts before, and their last end
    for (int64_t e0 = 0; e0 < p.experts; e0 += 64) {
        const int64_t e = e0 + lane;
        const PHX_GLOBAL int32_t *starts = (const PHX_GLOBAL int32_t *)p.starts;
        int64_t b = e < p.experts ? cut(starts[e], p.M) : 0;
        const int64_t next = e < p.experts ? cut(starts[e + 1], p.M) : 0;
        b = max(b, floor);
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int64_t o = __shfl_up(b, s);
            if (lane >= s) b = max(b, o);
        }
        const int64_t end = max(b, next), tiles = (end - b + TM - 1) / TM;
        int64_t sum = tiles;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int64_t o = __shfl_up(sum, s);
            if (lane >= s) sum += o;
        }
        const uint64_t has = __ballot(before + sum > wanted);
        if (has) {
            const int at = __builtin_ctzll(has);
            t.expert = e0 + at;
            t.m0 = __shfl(b + (wanted - before - (sum - tiles)) * TM, at);
            t.end = __shfl(end, at);
            t.live = true;
            return t;
        }
        before += __shfl(sum, 63);
        floor = __shfl(end, 63);
    }
    return t;
}

// The first form: a wave takes 16 columns by 16 rows, operands from memory.
__device__ __forceinline__ void gemm_f8(const PhxF8Gemm &p) {
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const uint32_t columns = (uint32_t)((p.N + 15) / 16);
    const Tile t = tile_of<16>(p, columns);
    if (!t.live) return;
    const int64_t n0 = (int64_t)t.column * 16, n = n0 + r, m = t.m0 + r;
    const uint32_t blocks = (uint32_t)((p.K + 127) / 128);
    int64_t row = m < t.end ? p.list ? ((const PHX_GLOBAL int32_t *)p.list)[m] : m : -1;
    if (row >= p.rows) row = -1;
    const PHX_GLOBAL char *a = (const PHX_GLOBAL char *)p.a + row * p.lda;
    const PHX_GLOBAL float *sa = (const PHX_GLOBAL float *)p.sa + row * p.lds;
    const PHX_GLOBAL char *w = (const PHX_GLOBAL char *)p.w + (t.expert * p.N + n) * p.K;
    const PHX_GLOBAL float *sw = (const PHX_GLOBAL float *)p.sw +
                                 (t.expert * ((p.N + 127) / 128) + n0 / 128) * blocks;
    phx_f4 acc = {0, 0, 0, 0};
    for (uint32_t b = 0; b < blocks; ++b) {
        phx_u4 x[2], y[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t k = (int64_t)b * 128 + 64 * h + 16 * g;
            x[h] = y[h] = (phx_u4){0, 0, 0, 0};
            if (k < p.K && n < p.N) x[h] = *(const PHX_GLOBAL phx_u4 *)(w + k);
            if (k < p.K && row >= 0) y[h] = *(const PHX_GLOBAL phx_u4 *)(a + k);
        }
        const v8i u = {(int)x[0][0], (int)x[0][1], (int)x[0][2], (int)x[0][3],
                       (int)x[1][0], (int)x[1][1], (int)x[1][2], (int)x[1][3]};
        const v8i v = {(int)y[0][0], (int)y[0][1], (int)y[0][2], (int)y[0][3],
                       (int)y[1][0], (int)y[1][1], (int)y[1][2], (int)y[1][3]};
        const phx_f4 sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            u, v, (phx_f4){0, 0, 0, 0}, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
        const float s = row >= 0 ? sa[b] * sw[b] : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(s, sum[i], acc[i]);
    }
    if (m >= t.end) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t c = n0 + 4 * g + i;
        if (c >= p.N) continue;
        float o = p.alpha * acc[i];
        const int64_t at = m * p.ldc + c;
        if (p.half) {
            PHX_GLOBAL _Float16 *to = (PHX_GLOBAL _Float16 *)p.c + at;
            if (p.beta != 0.0f) o = o + p.beta * (float)*to;
            *to = (_Float16)o;
        } else {
            PHX_GLOBAL float *to = (PHX_GLOBAL float *)p.c + at;
            if (p.beta != 0.0f) o = o + p.beta * *to;
            *to = o;
        }
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(64) void gemm_f8_first(PhxF8Gemm p) { gemm_f8(p); }
