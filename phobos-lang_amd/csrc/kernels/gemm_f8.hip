// Products of rows and weights in 8 bits, dense and grouped by expert (the layout
// and the arithmetic: include/phobos_hip.h, phx_gemm_f8 and phx_gemm_f8_grouped).
//
//   acc[m,n] = sum over blocks b of sa[m,b] sw[n/128,b] * sum over k in b of a[m,k] w[n,k]
//
// f16 outputs: the inner sum is one v_mfma_f32_16x16x128 of the codes. Of eight
// neighbouring products it keeps what is above 2^-13 of the largest (measured with
// one large and one small product; the sums of eight are added in f32): 1.4e-5 of an
// ordinary result's norm, where the rounding to f16 is 2.1e-4.
// Where large products cancel it shows. That is the price of twice the rate: f32
// outputs, which it would show in everywhere, take the codes as f16, exactly, and four
// v_mfma_f32_16x16x32: 1.1e-7, 8192 x 16384 x 8192 1860 us instead of 920.
// The inner sum is scaled and added in f32 by vector instructions, four for each
// 16 x 16, which run while the matrix cores work on the next one. The weights are the
// A operand, so that a lane holds neighbouring columns of one row of C, whose
// scales' product is one number.
//
// Large products: 8192 x 16384 x 8192, f16, 902-932 us (2360-2440 TFLOP/s; a library 8-bit
// product, with one scale for all, 660 to 800 with its inputs). The card is at its power
// limit, 1.8 GHz; of the cycles the matrix cores are busy 65 %, the vector instructions
// 48 %, LDS 29 %. A 256 x 256 tile alone on the chip, at 2.4 GHz, takes 1.18 us for 128 k
// and 0.76 without the 64 KiB that it loads into LDS for them; in the full chip 1.75 us.
// What is before and behind a tile's steps, 3 to 5 us, nothing hides where a CU holds one
// workgroup: it is a fifth of 16384 rows over 61 experts of 4096 x 2048, 208-214 us. There
// the groups' last tiles cost more still: of the 91 to 94 tiles of 256 rows 60 are not full
// and 22 to 30 hold 128 rows or fewer, so that 30 % of the rows worked on are none.
// Few rows are bound by the weights' bytes: 64 x 16384 x 8192 29.3 us (4.8 TB/s), 1 row
// 25.3 us (5.3 TB/s). Between them, where the tiles fill the GPU but once, it is the
// length of a step: 1000 x 1000 x 4144, f32, 17 us in 9 steps of 512 k; 384 x 16384 x 8192,
// f16, 70 us in 64 steps of 1.06 us on 192 CUs.
// (Also measured, at the same speed or slower: rows staged through registers instead of
// loaded into LDS directly; waves of 64 x 64 that read less LDS, as many or half as many,
// and one wave a SIMD of 128 x 64; loads spread over the whole step; a raised wave
// priority; 2 or 8 rows of tiles deep; the codes' conversions to f16 spread over the
// products of the tile before; W read ahead into L2 by a wave of its own; 256 columns of
// 16 for one row; results that change lanes, so that stores take whole rows: 2 % more for
// whole 16 bytes.)
#include <type_traits>

#include "f8.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void *lds_ptr;
typedef __attribute__((address_space(8))) void *rsrc_ptr;

constexpr uint32_t kNone = 0x80000000u;  // an offset past every resource's end: zeros

// Where a tile of TM rows lies: its expert, and C's rows from m0 up to end.
struct Tile {
    int64_t m0, end, expert;
    uint32_t column, rows;  // in tiles: its column, and the group's rows
    bool live;
};

// The same in every lane, and known to be.
__device__ __forceinline__ uint32_t uniform(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}

__device__ __forceinline__ uint32_t of_lane(uint32_t x, uint32_t lane) {
    return (uint32_t)__builtin_amdgcn_readlane((int)x, (int)lane);
}

// op over this lane's x and those of the lanes before it; 0 changes nothing.
template <typename Op>
__device__ __forceinline__ uint32_t upto(uint32_t x, Op op) {
    // within rows of 16 lanes, then the rows' last ones to the row behind, then the
    // lower half's last to the upper half
#define STEP(control, rows) \
    x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, control, rows, 0xf, false))
    STEP(0x111, 0xf);
    STEP(0x112, 0xf);
    STEP(0x114, 0xf);
    STEP(0x118, 0xf);
    STEP(0x142, 0xa);
    STEP(0x143, 0xc);
#undef STEP
    return x;
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
    uint32_t begin = 0, tiles = (uint32_t)((p.M + TM - 1) / TM), in;  // of the group; in it
    if (!p.starts) {
        in = uniform(phx_xcd_swizzle_any(blockIdx.x, gridDim.x));
    } else {
        const uint32_t lane = threadIdx.x & 63, E = (uint32_t)p.experts;
        const PHX_GLOBAL int32_t *starts = (const PHX_GLOBAL int32_t *)p.starts;
        auto at = [&](uint32_t e) { return (uint32_t)min(max(starts[min(e, E)], 0), (int32_t)p.M); };
        // 64 experts' first row and the one past the last, their tiles, and how many there
        // are up to each
        struct Range {
            uint32_t begin, end, tiles, upto;
        };
        auto range = [&](uint32_t e0, uint32_t floor, uint32_t before) {
            Range x;
            const uint32_t first = at(e0 + lane), last = at(e0 + lane + 1);
            x.begin = upto(max(first, floor), [](uint32_t a, uint32_t b) { return max(a, b); });
            x.end = e0 + lane < E ? max(x.begin, last) : x.begin;
            x.tiles = (x.end - x.begin + TM - 1) / TM;
            x.upto = before + upto(x.tiles, [](uint32_t a, uint32_t b) { return a + b; });
            return x;
        };
        Range x = range(0, 0, 0);
        uint32_t total = of_lane(x.upto, 63), floor = of_lane(x.end, 63);
        for (uint32_t e0 = 64; e0 < E; e0 += 64) {
            const Range y = range(e0, floor, total);
            floor = of_lane(y.end, 63);
            total = of_lane(y.upto, 63);
        }
        if (blockIdx.x >= total * columns) return t;
        const uint32_t id = uniform(phx_xcd_swizzle_any(blockIdx.x, total * columns));
        // (starts that are written while they are read, against what is asked for, may end
        // before this tile now: it is left out)
        uint32_t e0 = 0;
        while (of_lane(x.upto, 63) <= id / columns) {
            e0 += 64;
            if (e0 >= E) return t;
            x = range(e0, of_lane(x.end, 63), of_lane(x.upto, 63));
        }
        const uint32_t l = uniform(__builtin_ctzll(__ballot(x.upto > id / columns)));
        t.expert = uniform(e0 + l);
        begin = of_lane(x.begin, l);
        t.end = of_lane(x.end, l);
        tiles = of_lane(x.tiles, l);
        in = uniform(id - (of_lane(x.upto, l) - tiles) * columns);
    }
    const uint32_t top = in / (kDeep * columns) * kDeep, rest = in % (kDeep * columns);
    const uint32_t deep = min(tiles - top, kDeep);
    t.column = uniform(rest / deep);
    t.m0 = uniform(begin + (top + rest % deep) * TM);
    t.rows = tiles;
    t.live = true;
    return t;
}

// ------------------------------------------------------------------ tiles
// Where the tiles of WN x WM waves, each of NT x MT tiles of 16 columns by 16 rows,
// lie, and what their lanes load. WK such sets of waves take every WK-th block of K,
// each through its own part of LDS, and are added up at the end.
//
// A part holds 128 k: a row of W or of A is 128 bytes, its 16-byte chunk c at place
// c ^ f(row), so that the 16 rows of an operand's read touch every bank once.
// A lane's results of two neighbouring tiles of columns are eight neighbouring
// columns: the rows of W that the tiles 2i and 2i + 1 take interleave in fours.
template <int WN, int WM, int NT, int MT, int WK, int ST>
struct Shape {
    static constexpr uint32_t WAVES = WN * WM, TN = 16 * WN * NT, TM = 16 * WM * MT;
    static constexpr uint32_t PART = (TN + TM) * 128;
    // The rows' scales come four blocks at a time, a row's 16 bytes next to each other:
    // with four or eight sets, which take four or eight blocks a step, in its stage; with
    // fewer in places of their own, through registers (loaded into LDS directly, each read
    // of them would wait for the latest such load).
    static_assert(WK == 1 || WK == 2 || WK == 4 || WK == 8, "steps and fours of blocks");
    static constexpr bool STAGED = WK >= 4;
    static constexpr uint32_t ROWS = TM < 64 ? 64 : TM;       // that have a place
    static constexpr uint32_t SCALES = ROWS * (WK == 8 ? 32 : 16);
    static constexpr uint32_t S_LOADS = SCALES / 1024;  // waves that load them
    static constexpr uint32_t STAGE = PART * WK + (STAGED ? SCALES : 0);
    static constexpr uint32_t APART = STAGED ? 16 : 2 * SCALES;
    // How many tiles of columns before it is used W is read from LDS: four where there are
    // registers left for them (2048 x 4096 x 4096: up to 2 %).
    static constexpr int D = NT == 8 && MT == 2 ? 4 : 1;
    static constexpr uint32_t W_LOADS = TN / 8 / WAVES, A_LOADS = TM / 8 / WAVES;  // of 8 rows
    static_assert(TN % (8 * WAVES) == 0 && TM % (8 * WAVES) == 0, "whole loads a wave");
    static_assert(WK == 1 || TN * TM * 4 * (WK / 2) <= PART * WK, "the sums fit where the stages were");

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

// Stores a lane's eight columns of a row of C, which may start at any element: memory
// takes 16 bytes there too.
template <typename T>
__device__ __forceinline__ void store8(const PhxF8Gemm &p, const float (&acc)[8], int64_t m, int64_t n) {
    typedef T v8 __attribute__((ext_vector_type(8)));
    typedef v8 loose __attribute__((aligned(sizeof(T))));
    PHX_GLOBAL T *to = (PHX_GLOBAL T *)p.c + m * p.ldc + n;
    const bool whole = n + 8 <= p.N;
    v8 o;
    if (p.beta != 0.0f) {
        v8 old;
        if (whole)
            old = *(const PHX_GLOBAL loose *)to;
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) old[i] = n + i < p.N ? to[i] : (T)0;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (T)(p.alpha * acc[i] + p.beta * (float)old[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (T)(p.alpha * acc[i]);
    }
    // (between two dwords the 16 bytes take longer than a half, three dwords and a half:
    // 1475 x 13175 x 96 27.6 us, so 22.4, 13174 columns 18.8)
    if constexpr (sizeof(T) == 2) if (whole && ((uint64_t)to & 2)) {
        typedef T v6 __attribute__((ext_vector_type(6)));
        typedef uint32_t u3 __attribute__((ext_vector_type(3)));
        typedef u3 loose3 __attribute__((aligned(4)));
        to[0] = o[0];
        const v6 mid = {o[1], o[2], o[3], o[4], o[5], o[6]};
        *(PHX_GLOBAL loose3 *)(to + 1) = __builtin_bit_cast(u3, mid);
        to[7] = o[7];
        return;
    }
    if (whole)
        *(PHX_GLOBAL loose *)to = o;
    else
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (n + i < p.N) to[i] = o[i];
}

// Until at most LEFT of a wave's loads are on their way, and nothing to or from LDS.
template <uint32_t LEFT>
__device__ __forceinline__ void wait_for() {
    static_assert(LEFT < 64, "vmcnt's six bits");
    __builtin_amdgcn_s_waitcnt(0x0070 | (LEFT & 15) | (LEFT >> 4) << 14);
}

template <bool EXACT, int WN, int WM, int NT, int MT, int WK, int ST>
__device__ __forceinline__ void gemm_tile(const PhxF8Gemm &p, char *const (&st)[ST], char *sc) {
    using S = Shape<WN, WM, NT, MT, WK, ST>;
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const uint32_t all = uniform(threadIdx.x >> 6), wave = all % S::WAVES, wk = all / S::WAVES;
    const uint32_t wn = wave % WN, wm = wave / WN;
    const uint32_t columns = (uint32_t)((p.N + S::TN - 1) / S::TN);
    const Tile t = tile_of<S::TM>(p, columns);
    if (!t.live) return;
    const int64_t n0 = (int64_t)t.column * S::TN;
    const uint32_t blocks = (uint32_t)((p.K + 127) / 128);
    const uint32_t K = (uint32_t)p.K;
    // Of few rows every workgroup reads weights of its own, all at the same k at the same
    // time, rows of W apart, which memory is slower with than it need be: they start
    // at different blocks instead and go round (in fours, as the scales come). 64 x 16384
    // x 8192: 31 us, all from the first on 35; 1 x 16384 x 8192: 29.8 and 32.4; f32, 40 rows
    // over 14 experts of 2048 x 4096: 30.4 and 32.5. (With more rows neighbours share what
    // they read: 256 x 256 tiles would take 1 to 4 % longer so.)
    constexpr bool TURNS = S::TM <= 64;
    const uint32_t turn = !TURNS || t.rows > kDeep || blocks % 4 ? 0 : t.column * 12 % blocks;
    auto turned = [&](uint32_t b) {
        return b >= blocks ? b : b + turn >= blocks ? b + turn - blocks : b + turn;
    };

    // W: rows of this tile up to N's end
    const int64_t left_n = min(p.N - n0, (int64_t)S::TN);
    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(p.w + (t.expert * p.N + n0) * p.K), 0, (int)(left_n * p.K), 0x00020000);
    // A: the tile's rows, or with a list all of them
    const int64_t base = p.list ? 0 : t.m0, left_m = min(t.end - t.m0, (int64_t)S::TM);
    const int64_t rows = p.list ? max(p.rows, (int64_t)1) : left_m;  // (none: nothing is read)
    const __amdgpu_buffer_rsrc_t ar = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(p.a + base * p.lda), 0, (int)((rows - 1) * p.lda + p.K), 0x00020000);
    const __amdgpu_buffer_rsrc_t sr = __builtin_amdgcn_make_buffer_rsrc(
        (void *)(p.sa + base * p.lds * 4), 0, (int)(rows * p.lds * 4), 0x00020000);
    // the rows of this wave's loads, and the entries of the list that say where they are
    auto a_row = [&](uint32_t i) {
        return i < S::A_LOADS ? (wave * S::A_LOADS + i) * 8 + lane / 8 : all * 64 % S::ROWS + lane;
    };
    int32_t entry[S::A_LOADS + 1];
    if (p.list) {
#pragma unroll
        for (uint32_t i = 0; i <= S::A_LOADS; ++i)
            entry[i] = ((const PHX_GLOBAL int32_t *)p.list)[t.m0 + min((int64_t)a_row(i), left_m - 1)];
    }
    // the i-th's row in A, or none
    auto source = [&](uint32_t i) -> int64_t {
        if (a_row(i) >= left_m) return -1;
        if (!p.list) return a_row(i);
        return entry[i] >= 0 && entry[i] < p.rows ? entry[i] : -1;
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
    auto find_rows = [&]() {
#pragma unroll
        for (uint32_t i = 0; i < S::A_LOADS; ++i) {
            const int64_t at = source(i);
            a_off[i] = at < 0 ? kNone : (uint32_t)(at * p.lda) + a_k(i);
        }
        if (all < S::S_LOADS) {
            const int64_t at = source(S::A_LOADS);
            s_off = at < 0 ? kNone : (uint32_t)(at * p.lds * 4);
        }
    };
    // Of block b the chunks behind K's end are nowhere: they stay so, as nothing but what
    // lies behind it is loaded after the last block. (Where W's blocks go round each load
    // looks by itself: 2 to 3 % of a step's time.)
    auto cut = [&](uint32_t b) {
        if (TURNS || b * 128 + 128 <= K) return;
#pragma unroll
        for (uint32_t i = 0; i < S::W_LOADS; ++i)
            if (b * 128 + w_k(i) >= K) w_off[i] = kNone;
#pragma unroll
        for (uint32_t i = 0; i < S::A_LOADS; ++i)
            if (b * 128 + a_k(i) >= K) a_off[i] = kNone;
    };
    // the i-th of this wave's loads of block b: 8 rows of W or of A
    auto load = [&](char *stage, uint32_t b, uint32_t i) {
        const uint32_t k = turned(b) * 128;
        char *to = stage + wk * S::PART;
        if (i < S::W_LOADS) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                wr, (lds_ptr)(to + (wave * S::W_LOADS + i) * 1024), 16,
                TURNS && k + w_k(i) >= K ? kNone : w_off[i], (int)k, 0, 0);
        } else {
            const uint32_t j = i - S::W_LOADS;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                ar, (lds_ptr)(to + S::TN * 128 + (wave * S::A_LOADS + j) * 1024), 16,
                TURNS && k + a_k(j) >= K ? kNone : a_off[j], (int)k, 0, 0);
        }
    };
    // the scales of the tile's rows of the four blocks from b on: where this wave's share
    // is (behind the rows' end nowhere), and into LDS
    auto scales_at = [&](uint32_t b) { return b < (uint32_t)p.lds ? s_off : kNone; };
    auto load_scales = [&](char *to, uint32_t b) {
        b = turned(b + all * 64 / S::ROWS * 4);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(sr, (lds_ptr)(to + all * 1024), 16, scales_at(b),
                                                 (int)(b * 4), 0, 0);
    };
    // the weights' scales of 64 blocks, one a lane
    const PHX_GLOBAL float *sw = (const PHX_GLOBAL float *)p.sw +
                                 (t.expert * ((p.N + 127) / 128) +
                                  min((n0 + wn * (16 * NT)) / 128, (p.N - 1) / 128)) * blocks;
    float w_scales;
    auto load_w_scales = [&](uint32_t b) { w_scales = sw[min(turned(b + lane), blocks - 1)]; };

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

    constexpr int D = S::D;
    using C = Codes<EXACT>;
    C x[MT];                 // this step's rows
    phx_u4 w_next[D][2];     // the next tiles of columns
    phx_u4 x_next[MT][2];    // the next step's rows
    float f[MT], f_next[MT], f_last[MT];
    phx_f4 sum[MT];
    auto read_w = [&](const char *stage, int n) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            w_next[n % D][h] = *(const phx_u4 *)(stage + wk * S::PART + w_at[n % 2][h] + n / 2 * 4096);
    };
    auto read_x = [&](const char *stage, int m) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            x_next[m][h] = *(const phx_u4 *)(stage + wk * S::PART + a_at[h] + m * 2048);
    };
    auto read_scale = [&](const char *stage, uint32_t b0, int m) {
        const char *from = S::STAGED ? stage + WK * S::PART + wk / 4 * (S::ROWS * 16)
                                     : sc + b0 / 4 % 2 * S::SCALES;
        return *(const float *)(from + s_at + m * 256 + (b0 + wk) % 4 * 4);
    };

    // A step: while its tiles are multiplied, the sums of the tile before are scaled, the
    // next tile's weights read from LDS, and the blocks of ST - 1 steps ahead loaded
    // into the stage of the step before. In its last D columns of tiles, where nothing
    // of its stage is left to read, comes the one barrier: a wave's own loads of the
    // next stage have landed before it, every wave's behind it, and behind it the
    // next step's rows are read as this one's are used up. (Behind the last block
    // the loads are of nothing, into what nobody reads.)
    constexpr uint32_t AHEAD = ST - 1, EACH = S::W_LOADS + S::A_LOADS;
    constexpr uint32_t SLOTS = (NT - D) * MT, PER_SLOT = (EACH + SLOTS - 1) / SLOTS;
    const bool loads_scales = all < S::S_LOADS;
    phx_u4 scales = {0, 0, 0, 0};
    auto pass = [&]() {
        if (S::STAGED && loads_scales)
            wait_for<(AHEAD - 1) * (EACH + 1)>();
        else
            wait_for<(AHEAD - 1) * EACH>();
        asm volatile("" ::: "memory");  // no access moves across
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    load_w_scales(0);
    // what a step loads besides its tiles' blocks
    auto load_more = [&](uint32_t b0, char *fill) {
        if (!loads_scales) return;
        if (S::STAGED) {
            load_scales(fill + WK * S::PART, b0 + AHEAD * WK);
            return;
        }
        // the next four blocks' scales: loaded at the first of these four, written at the
        // third (at the two steps of the four, where a step takes two), behind two
        // barriers or more since what was there was read
        if (b0 % 4 == 0) {
            const uint32_t b = turned(b0 + 4);
            scales = __builtin_bit_cast(
                phx_u4, __builtin_amdgcn_raw_buffer_load_b128(sr, scales_at(b), (int)(b * 4), 0));
        }
        if (b0 % 4 == 2)
            *(phx_u4 *)(sc + (b0 / 4 + 1) % 2 * S::SCALES + threadIdx.x * 16) = scales;
    };
    auto step = [&](uint32_t b0, char *now, char *then, char *fill) {
        const uint32_t b = b0 + wk;
        const float scale =
            __builtin_bit_cast(float, of_lane(__builtin_bit_cast(uint32_t, w_scales), b % 64));
        if (b0 % 64 == 64 - WK) load_w_scales(b0 + WK);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            x[m].of(x_next[m][0], x_next[m][1]);
            f_last[m] = f[m];
            f[m] = f_next[m] * scale;
            if (WK > 1) f[m] = b < blocks ? f[m] : 0.0f;
        }
        load_more(b0, fill);
        cut(b + AHEAD * WK);
        C w;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            w.of(w_next[n % D][0], w_next[n % D][1]);
            if (n + D < NT) read_w(now, n + D);
            const int done = n ? n - 1 : NT - 1;
#pragma unroll
            for (int j = 0; j < C::STEPS; ++j)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    if (j == 0) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[done][m][i] =
                                __builtin_fmaf(n ? f[m] : f_last[m], sum[m][i], acc[done][m][i]);
                        // (here, and not behind the branches of a later step)
                        asm volatile("" : "+v"(acc[done][m]));
                    }
                    sum[m] = C::product(w, x[m], j, j ? sum[m] : (phx_f4){0, 0, 0, 0});
                    if (j == 0) {
                        const uint32_t slot = n * MT + m;
#pragma unroll
                        for (uint32_t i = slot * PER_SLOT; i < (slot + 1) * PER_SLOT; ++i)
                            if (i < EACH) load(fill, b + AHEAD * WK, i);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    if (n >= NT - D && j == 0) {
                        if (n == NT - D && m == 0) pass();
                        if (m == 0) read_w(then, n - (NT - D));
                        if (n == NT - D) {
                            read_x(then, m);
                            f_next[m] = read_scale(then, b0 + WK, m);
                        }
                    }
                }
        }
    };
    // (the first weights before A's rows are looked up in the list)
    cut(wk);
#pragma unroll
    for (uint32_t i = 0; i < S::W_LOADS; ++i) load(st[0], wk, i);
    find_rows();
    if (!S::STAGED && loads_scales) load_scales(sc, 0);
#pragma unroll
    for (uint32_t u = 0; u < AHEAD; ++u) {
        cut(u * WK + wk);
        if (S::STAGED && loads_scales) load_scales(st[u] + WK * S::PART, u * WK);
#pragma unroll
        for (uint32_t i = u ? 0 : S::W_LOADS; i < EACH; ++i) load(st[u], u * WK + wk, i);
    }
    pass();
#pragma unroll
    for (int n = 0; n < D; ++n) read_w(st[0], n);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        read_x(st[0], m);
        f_next[m] = read_scale(st[0], 0, m);
        f[m] = 0.0f;
        sum[m] = (phx_f4){0, 0, 0, 0};
    }
    auto steps = [&](auto one) {
        uint32_t b = 0;
        for (; b + AHEAD * WK < blocks; b += ST * WK)
#pragma unroll
            for (int u = 0; u < ST; ++u)
                one(b + u * WK, st[u], st[(u + 1) % ST], st[(u + ST - 1) % ST]);
#pragma unroll
        for (int u = 0; u < ST - 1; ++u)
            if (b + u * WK < blocks) one(b + u * WK, st[u], st[(u + 1) % ST], st[(u + ST - 1) % ST]);
    };
    // (of a last tile of rows few may be left: waves without one load and pass on)
    if (WM == 1 || wm * (16 * MT) < left_m)
        steps(step);
    else
        steps([&](uint32_t b0, char *, char *, char *fill) {
            load_more(b0, fill);
            cut(b0 + wk + AHEAD * WK);
#pragma unroll
            for (uint32_t i = 0; i < EACH; ++i) load(fill, b0 + wk + AHEAD * WK, i);
            pass();
        });
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            acc[NT - 1][m][i] = __builtin_fmaf(f[m], sum[m][i], acc[NT - 1][m][i]);
    // (the loads behind the last block write zeros: before the sums, and before LDS is
    // another workgroup's)
    wait_for<0>();
    if (WK > 1) {
        // the sets' sums to LDS; of them each wave adds up and stores its share
        __syncthreads();
        constexpr uint32_t SUM = S::TN * S::TM * 4;
        auto at = [&](uint32_t set, uint32_t n, uint32_t m) {
            char *half = set < WK / 2 ? st[0] + set * SUM : st[1] + (set - WK / 2) * SUM;
            return (phx_f4 *)(half + ((wave * NT + n) * MT + m) * 1024 + lane * 16);
        };
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < MT; ++m) *at(wk, n, m) = acc[n][m];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                if (((uint32_t)(n / 2 * MT + m)) % WK != wk) continue;
                acc[n][m] = *at(0, n, m);
#pragma unroll
                for (int set = 1; set < WK; ++set) acc[n][m] = acc[n][m] + *at(set, n, m);
            }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const uint32_t row = wm * (16 * MT) + 16 * m + r;
        if (row >= left_m) continue;
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            if (WK > 1 && ((uint32_t)(n / 2 * MT + m)) % WK != wk) continue;
            const float o[8] = {acc[n][m][0], acc[n][m][1], acc[n][m][2], acc[n][m][3],
                                acc[n + 1][m][0], acc[n + 1][m][1], acc[n + 1][m][2], acc[n + 1][m][3]};
            const int64_t c = n0 + wn * (16 * NT) + 16 * n + 8 * g;
            if (c < p.N) store8<std::conditional_t<EXACT, float, _Float16>>(p, o, t.m0 + row, c);
        }
    }
}

}  // namespace

#define STAGES_2(S) s0[S::STAGE / 16], s1[S::STAGE / 16]
#define STAGES_3(S) STAGES_2(S), s2[S::STAGE / 16]
#define STAGES_4(S) STAGES_3(S), s3[S::STAGE / 16]
#define LIST_2 (char *)s0, (char *)s1
#define LIST_3 LIST_2, (char *)s2
#define LIST_4 LIST_3, (char *)s3
// (each stage is an array of its own, so that the compiler sees that what is read and
// what is being filled differ)
#define TILE(EXACT, suffix, WN, WM, NT, MT, WK, ST)                                             \
    extern "C" __global__ __launch_bounds__(64 * WN * WM * WK) void                             \
        gemm_f8_##suffix##_##WN##x##WM##_##NT##x##MT##_k##WK##_s##ST(PhxF8Gemm p) {             \
        using S = Shape<WN, WM, NT, MT, WK, ST>;                                                \
        __shared__ phx_u4 STAGES_##ST(S), sc[S::APART / 16];                                    \
        char *const st[ST] = {LIST_##ST};                                                       \
        gemm_tile<EXACT, WN, WM, NT, MT, WK, ST>(p, st, (char *)sc);                            \
    }
#define BOTH(WN, WM, NT, MT, WK, ST)                                                            \
    TILE(false, f16, WN, WM, NT, MT, WK, ST)                                                    \
    TILE(true, f32, WN, WM, NT, MT, WK, ST)
TILE(false, f16, 1, 1, 2, 1, 4, 4)
BOTH(1, 1, 2, 1, 4, 2)
TILE(true, f32, 1, 1, 2, 1, 8, 3)
TILE(false, f16, 2, 1, 2, 1, 4, 3)
BOTH(2, 1, 2, 2, 2, 3)
TILE(false, f16, 2, 2, 2, 2, 2, 4)
TILE(true, f32, 1, 2, 4, 2, 4, 2)
BOTH(2, 2, 2, 2, 1, 4)
BOTH(2, 2, 4, 2, 1, 3)
TILE(true, f32, 2, 2, 4, 4, 1, 2)
TILE(false, f16, 2, 4, 8, 2, 1, 3)
TILE(false, f16, 2, 4, 8, 4, 1, 2)
