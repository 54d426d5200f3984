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

// The same in every lane, and known to be.
__device__ __forceinline__ uint32_t uniform(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}

__device__ __forceinline__ uint32_t of_lane(uint32_t x, uint32_t lane) {
    return (uint32_t)__builtin_amdgcn_readlane((int)x, (int)lane);
}

// Tiles of the groups in their order, `columns` of them for every TM rows. The groups'
// ranges are made to ascend, so that none overlap whatever the starts hold.
//
// The workgroups of an XCD take neighbouring tiles, up to kDeep of one column next to
// each other, so that they share rows and weights in its L2.
constexpr uint32_t kDeep = 4;

template <int TM>
__device__ __forceinline__ Tile tile_of(const PhxF8Gemm &p, uint32_t columns) {
    Tile t;
    t.live = false;
    t.expert = 0;
    t.end = p.M;
    uint32_t tiles = (uint32_t)((p.M + TM - 1) / TM), first = 0, id;
    int64_t begin = 0;
    if (!p.starts) {
        id = phx_xcd_swizzle_any(blockIdx.x, gridDim.x);
    } else {
        const uint32_t lane = threadIdx.x & 63, E = (uint32_t)p.experts, M = (uint32_t)p.M;
        const PHX_GLOBAL int32_t *starts = (const PHX_GLOBAL int32_t *)p.starts;
        auto at = [&](uint32_t e) { return (uint32_t)min(max(starts[min(e, E)], 0), (int32_t)M); };
        // 64 experts' first and last row, and how many tiles there are up to each
        struct Range {
            uint32_t begin, end, tiles, upto;
        };
        auto range = [&](uint32_t e0, uint32_t floor, uint32_t before) {
            Range x;
            x.begin = max(at(e0 + lane), floor);
#pragma unroll
            for (int s = 1; s < 64; s <<= 1) {
                const uint32_t o = __shfl_up(x.begin, s);
                if (lane >= s) x.begin = max(x.begin, o);
            }
            x.end = e0 + lane < E ? max(x.begin, at(e0 + lane + 1)) : x.begin;
            x.tiles = (x.end - x.begin + TM - 1) / TM;
            x.upto = x.tiles;
#pragma unroll
            for (int s = 1; s < 64; s <<= 1) {
                const uint32_t o = __shfl_up(x.upto, s);
                if (lane >= s) x.upto += o;
            }
            x.upto += before;
            return x;
        };
        Range x = range(0, 0, 0);
        uint32_t total = of_lane(x.upto, 63);
        if (E > 64) {
            uint32_t floor = of_lane(x.end, 63);
            for (uint32_t e0 = 64; e0 < E; e0 += 64) {
                const Range y = range(e0, floor, total);
                floor = of_lane(y.end, 63);
                total = of_lane(y.upto, 63);
            }
        }
        if (blockIdx.x >= total * columns) return t;
        id = phx_xcd_swizzle_any(blockIdx.x, total * columns);
        const uint32_t wanted = id / columns;
        uint32_t e0 = 0;
        while (of_lane(x.upto, 63) <= wanted) {
            e0 += 64;
            x = range(e0, of_lane(x.end, 63), of_lane(x.upto, 63));
        }
        const uint32_t l = uniform(__builtin_ctzll(__ballot(x.upto > wanted)));
        t.expert = e0 + l;
        t.expert = uniform((uint32_t)t.expert);
        begin = of_lane(x.begin, l);
        t.end = of_lane(x.end, l);
        tiles = of_lane(x.tiles, l);
        first = of_lane(x.upto, l) - tiles;
    }
    id = uniform(id);
    const uint32_t in = id - first * columns;
    const uint32_t top = in / (kDeep * columns) * kDeep, rest = in % (kDeep * columns);
    const uint32_t deep = min(tiles - top, kDeep);
    t.column = uniform(rest / deep);
    t.m0 = uniform((uint32_t)begin + (top + rest % deep) * TM);
    t.live = true;
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
            u, v, (phx_f4){0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
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

// ------------------------------------------------------------------ tiles
// Where the tiles of WN x WM waves, each of NT x MT tiles of 16 columns by 16 rows,
// lie, and what their lanes load.
//
// A stage holds 128 k: a row of W or of A is 128 bytes, its 16-byte chunk c at place
// c ^ f(row), so that the 16 rows of an operand's read touch every bank once.
// A lane's results of two neighbouring tiles of columns are eight neighbouring
// columns: the rows of W that the tiles 2i and 2i + 1 take interleave in fours.
template <int WN, int WM, int NT, int MT>
struct Shape {
    static constexpr uint32_t WAVES = WN * WM, TN = 16 * WN * NT, TM = 16 * WM * MT;
    static constexpr uint32_t STAGE = (TN + TM) * 128;
    static constexpr uint32_t W_LOADS = TN / 8 / WAVES, A_LOADS = TM / 8 / WAVES;  // of 8 rows
    static_assert(TN % (8 * WAVES) == 0 && TM % (8 * WAVES) == 0, "whole loads a wave");

    static __device__ __forceinline__ uint32_t w_row(uint32_t tile, uint32_t r) {
        return 32 * (tile / 2) + 8 * (r / 4) + 4 * (tile % 2) + r % 4;
    }
    static __device__ __forceinline__ uint32_t w_swizzle(uint32_t row) {
        return (row >> 1 & 1) | (row >> 3 & 3) << 1;
    }
    static __device__ __forceinline__ uint32_t a_swizzle(uint32_t row) { return row >> 1 & 7; }
};

// A lane's 32 codes of an operand, and what multiplies them.
template <bool EXACT>
struct Codes;
template <>
struct Codes<false> {
    static constexpr int STEPS = 1;
    v8i v;
    __device__ __forceinline__ void of(phx_u4 x, phx_u4 y) {
        v = (v8i){(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
    }
    static __device__ __forceinline__ phx_f4 product(const Codes &w, const Codes &x, int, phx_f4 c) {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, c, 0, 0, 0, 0, 0, 0);
    }
};
template <>
struct Codes<true> {
    static constexpr int STEPS = 4;
    phx_h8 v[4];
    __device__ __forceinline__ void of(phx_u4 x, phx_u4 y) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            phx_u4 h;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t c = j < 2 ? x[2 * j + i / 2] : y[2 * (j - 2) + i / 2];
                h[i] = __builtin_bit_cast(uint32_t, i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, true)
                                                          : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, false));
            }
            v[j] = __builtin_bit_cast(phx_h8, h);
        }
    }
    static __device__ __forceinline__ phx_f4 product(const Codes &w, const Codes &x, int j, phx_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[j], x.v[j], c, 0, 0, 0);
    }
};

// Stores a lane's eight columns of a row of C.
__device__ __forceinline__ void store8(const PhxF8Gemm &p, const float (&acc)[8], int64_t m, int64_t n) {
    const int64_t at = m * p.ldc + n;
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = p.alpha * acc[i];
    if (p.half) {
        PHX_GLOBAL _Float16 *to = (PHX_GLOBAL _Float16 *)p.c + at;
        if (p.wide && n + 8 <= p.N) {
            phx_h8 h;
            if (p.beta != 0.0f) {
                h = *(PHX_GLOBAL phx_h8 *)to;
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = o[i] + p.beta * (float)h[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = (_Float16)o[i];
            *(PHX_GLOBAL phx_h8 *)to = h;
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (n + i < p.N) {
                if (p.beta != 0.0f) o[i] = o[i] + p.beta * (float)to[i];
                to[i] = (_Float16)o[i];
            }
        return;
    }
    PHX_GLOBAL float *to = (PHX_GLOBAL float *)p.c + at;
    if (p.wide && n + 8 <= p.N) {
        phx_f4 v[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v[h] = (phx_f4){o[4 * h], o[4 * h + 1], o[4 * h + 2], o[4 * h + 3]};
            if (p.beta != 0.0f) v[h] = v[h] + p.beta * ((PHX_GLOBAL phx_f4 *)to)[h];
        }
        ((PHX_GLOBAL phx_f4 *)to)[0] = v[0];
        ((PHX_GLOBAL phx_f4 *)to)[1] = v[1];
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (n + i < p.N) {
            if (p.beta != 0.0f) o[i] = o[i] + p.beta * to[i];
            to[i] = o[i];
        }
}

template <bool EXACT, int WN, int WM, int NT, int MT>
__device__ __forceinline__ void gemm_tile(const PhxF8Gemm &p, char *s0, char *s1, char *sc) {
    using S = Shape<WN, WM, NT, MT>;
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wn = wave % WN, wm = wave / WN;
    const uint32_t columns = (uint32_t)((p.N + S::TN - 1) / S::TN);
    const Tile t = tile_of<S::TM>(p, columns);
    if (!t.live) return;
    const int64_t n0 = (int64_t)t.column * S::TN;
    const uint32_t blocks = (uint32_t)((p.K + 127) / 128);
    const uint32_t K = (uint32_t)p.K;

    // W: rows of this tile up to N's end
    const int64_t left_n = min(p.N - n0, (int64_t)S::TN);
    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(p.w + (t.expert * p.N + n0) * p.K), 0, (int)(left_n * p.K), 0x00020000);
    // A: the tile's rows, or with a list all of them
    const int64_t base = p.list ? 0 : t.m0, left_m = min(t.end - t.m0, (int64_t)S::TM);
    const int64_t rows = p.list ? p.rows : left_m;
    const __amdgpu_buffer_rsrc_t ar = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(p.a + base * p.lda), 0, (int)((rows - 1) * p.lda + p.K), 0x00020000);
    const __amdgpu_buffer_rsrc_t sr = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(p.sa + base * p.lds * 4), 0, (int)(rows * p.lds * 4), 0x00020000);
    // a row of the tile in A, or none
    auto source = [&](uint32_t row) -> int64_t {
        if (row >= left_m) return -1;
        if (!p.list) return row;
        const int64_t i = ((const PHX_GLOBAL int32_t *)p.list)[t.m0 + row];
        return i >= 0 && i < p.rows ? i : -1;
    };
    // the k of a lane's chunk in a load's row
    auto w_k = [&](uint32_t i) {
        return (lane % 8 ^ S::w_swizzle((wave * S::W_LOADS + i) * 8 + lane / 8)) * 16;
    };
    auto a_k = [&](uint32_t i) {
        return (lane % 8 ^ S::a_swizzle((wave * S::A_LOADS + i) * 8 + lane / 8)) * 16;
    };
    uint32_t w_off[S::W_LOADS], a_off[S::A_LOADS], s_off = kNone;
#pragma unroll
    for (uint32_t i = 0; i < S::W_LOADS; ++i) {
        const uint32_t row = (wave * S::W_LOADS + i) * 8 + lane / 8;
        w_off[i] = row * K + w_k(i);  // (rows past N's end lie past the resource's)
    }
#pragma unroll
    for (uint32_t i = 0; i < S::A_LOADS; ++i) {
        const uint32_t row = (wave * S::A_LOADS + i) * 8 + lane / 8;
        const int64_t at = source(row);
        a_off[i] = at < 0 ? kNone : (uint32_t)(at * p.lda) + a_k(i);
    }
    {
        const int64_t at = source(threadIdx.x % S::TM);
        s_off = at < 0 ? kNone : (uint32_t)(at * p.lds * 4);
    }
    auto load = [&](char *to, uint32_t b) {
        const uint32_t k = b * 128;
#pragma unroll
        for (uint32_t i = 0; i < S::W_LOADS; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                wr, (lds_ptr)(to + (wave * S::W_LOADS + i) * 1024), 16,
                k + w_k(i) < K ? w_off[i] : kNone, (int)k, 0, 0);
#pragma unroll
        for (uint32_t i = 0; i < S::A_LOADS; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                ar, (lds_ptr)(to + S::TN * 128 + (wave * S::A_LOADS + i) * 1024), 16,
                k + a_k(i) < K ? a_off[i] : kNone, (int)k, 0, 0);
    };
    // four blocks' scales of the tile's rows at a time (waves that are more than the
    // rows take load what others load, to the same place)
    auto load_scales = [&](uint32_t b) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            sr, (lds_ptr)(sc + (b / 4 % 2) * (S::TM * 16) + wave % (S::TM / 64) * 1024), 16, s_off,
            (int)(b * 4), 0, 0);
    };
    const __attribute__((address_space(4))) float *sw =
        (const __attribute__((address_space(4))) float *)p.sw +
        (t.expert * ((p.N + 127) / 128) +
         min((n0 + wn * (16 * NT)) / 128, (p.N - 1) / 128)) * blocks;

    phx_f4 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[n][m] = (phx_f4){0, 0, 0, 0};

    // where a lane's operands lie in a stage
    uint32_t w_at[2][2], a_at[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
            const uint32_t row = S::w_row(odd, r);  // (the swizzle repeats every 32 rows)
            w_at[odd][h] = (wn * (16 * NT) + row) * 128 + ((g + 4 * h) ^ S::w_swizzle(row)) * 16;
        }
        a_at[h] = (S::TN + wm * (16 * MT) + r) * 128 + ((g + 4 * h) ^ S::a_swizzle(r)) * 16;
    }
    const uint32_t s_at = (wm * (16 * MT) + r) * 16;

    auto multiply = [&](const char *from, uint32_t b, float scale) {
        using C = Codes<EXACT>;
        C x[MT], w;
        float f[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            x[m].of(*(const phx_u4 *)(from + a_at[0] + m * 2048),
                    *(const phx_u4 *)(from + a_at[1] + m * 2048));
            f[m] = *(const float *)(sc + (b / 4 % 2) * (S::TM * 16) + s_at + m * 256 + b % 4 * 4) * scale;
        }
        // a tile's sum is scaled while the next tiles are multiplied
        phx_f4 sum[MT];
        phx_u4 next[2];
        auto read = [&](int n) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                next[h] = *(const phx_u4 *)(from + w_at[n % 2][h] + n / 2 * 4096);
        };
        read(0);
#pragma unroll
        for (int n = 0; n <= NT; ++n) {
            if (n < NT) w.of(next[0], next[1]);
            if (n + 1 < NT) read(n + 1);
#pragma unroll
            for (int j = 0; j < C::STEPS; ++j)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    if (n > 0 && j == 0) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[n - 1][m][i] = __builtin_fmaf(f[m], sum[m][i], acc[n - 1][m][i]);
                        // (here, and not behind the branches of a later step)
                        asm volatile("" : "+v"(acc[n - 1][m]));
                    }
                    if (n < NT) sum[m] = C::product(w, x[m], j, j ? sum[m] : (phx_f4){0, 0, 0, 0});
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    };
    // One barrier a step: before it a wave's own loads of this step's stage have
    // landed, and behind it every wave's have, and all reads of the other stage are
    // done, which the next step's loads then fill.
    load_scales(0);
    load(s0, 0);
    float scale = sw[0];
    auto step = [&](uint32_t b, char *now, char *next) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        const float f = scale;
        // (behind the last block the loads are of nothing, into what nobody reads)
        if ((b + 1) % 4 == 0) load_scales(b + 1);
        load(next, b + 1);
        scale = sw[min(b + 1, blocks - 1)];
        __builtin_amdgcn_sched_barrier(0);
        multiply(now, b, f);
    };
    uint32_t b = 0;
    for (; b + 2 <= blocks; b += 2) {
        step(b, s0, s1);
        step(b + 1, s1, s0);
    }
    if (b < blocks) step(b, s0, s1);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const uint32_t row = wm * (16 * MT) + 16 * m + r;
        if (row >= left_m) continue;
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            const float o[8] = {acc[n][m][0], acc[n][m][1], acc[n][m][2], acc[n][m][3],
                                acc[n + 1][m][0], acc[n + 1][m][1], acc[n + 1][m][2], acc[n + 1][m][3]};
            const int64_t c = n0 + wn * (16 * NT) + 16 * n + 8 * g;
            if (c < p.N) store8(p, o, t.m0 + row, c);
        }
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(64) void gemm_f8_first(PhxF8Gemm p) { gemm_f8(p); }

#define TILE(EXACT, suffix, WN, WM, NT, MT)                                                     \
    extern "C" __global__ __launch_bounds__(64 * WN * WM) __attribute__((amdgpu_waves_per_eu(2))) void \
        gemm_f8_##suffix##_##WN##x##WM##_##NT##x##MT(PhxF8Gemm p) {                             \
        using S = Shape<WN, WM, NT, MT>;                                                        \
        __shared__ phx_u4 s0[S::STAGE / 16], s1[S::STAGE / 16], sc[2 * S::TM];                  \
        gemm_tile<EXACT, WN, WM, NT, MT>(p, (char *)s0, (char *)s1, (char *)sc);                \
    }
TILE(false, f16, 2, 4, 8, 4)
TILE(false, f16, 2, 2, 4, 4)
TILE(true, f32, 2, 2, 4, 4)
