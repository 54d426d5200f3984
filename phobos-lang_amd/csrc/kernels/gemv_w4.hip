// C = alpha*A@W + beta*C for up to 64 rows of A and 4-bit weights W with a
// scale and a zero point per group of K (the layout and the arithmetic:
// include/phobos_hip.h, phx_gemv_w4).
//
//   acc[m,n] = sum over groups g of s[g,n] * sum over k in g of a[m,k] (q[k,n] - z[g,n])
//
// The inner sum is in f32 of exact products, scaled in f32.
//
// The codes less their zero points are the matrix operand, as f16 (or bf16 with
// f32 rows in three bf16 terms): a tile's dword is a lane's eight k of
// v_mfma_f32_16x16x32, so 16 bytes of a lane are four products' operands, and a
// group is one to four of them, whose sum is scaled once.
#include "phx_common.h"
#include "phx_decode.h"

#define PHX_GLOBAL __attribute__((address_space(1)))

// Codes [K, N], one a byte, into the packed tiles; a thread per dword.
extern "C" __global__ __launch_bounds__(256) void w4_pack(const uint8_t *codes, uint32_t *packed,
                                                          int64_t N, int64_t K, int64_t words) {
    const int64_t kb = (K + PHX_W4_TILE_K - 1) / PHX_W4_TILE_K;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words;
         i += (int64_t)gridDim.x * 256) {
        const int64_t tile = i >> 8;
        const int j = i & 3, r = (i >> 2) & 15, q = (i >> 6) & 3;
        const int64_t n = tile / kb * 16 + r, k0 = tile % kb * 128 + 32 * j + 8 * q;
        uint32_t word = 0;
        for (int e = 0; e < 8; ++e)
            if (n < N && k0 + e < K)
                word |= (uint32_t)(codes[(k0 + e) * N + n] & 15) << (4 * (e / 2 + 4 * (e % 2)));
        packed[i] = word;
    }
}

namespace {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ uint32_t in_vgpr(uint32_t x) {
    asm("" : "+v"(x));
    return x;
}

// 16 rows by 32 k of A as a matrix operand (a lane: row lane % 16, eight k from
// 8 (lane / 16) on), rows and k that do not exist as zeros: one f16 term, or
// three bf16 terms of an f32, which hold its 24 bits.
template <typename T>
struct Rows;
template <>
struct Rows<_Float16> {
    phx_h8 v;
};
template <>
struct Rows<float> {
    b8 v[3];
};

__device__ __forceinline__ void load(Rows<_Float16> &r, __amdgpu_buffer_rsrc_t a, uint32_t off) {
    r.v = __builtin_bit_cast(phx_h8, __builtin_amdgcn_raw_buffer_load_b128(a, off, 0, 0));
}
__device__ __forceinline__ void load(Rows<float> &r, __amdgpu_buffer_rsrc_t a, uint32_t off) {
    const phx_u4 x = __builtin_amdgcn_raw_buffer_load_b128(a, off, 0, 0);
    const phx_u4 y = __builtin_amdgcn_raw_buffer_load_b128(a, off, 16, 0);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        // the top 16 bits, what they leave, and what that leaves: each exact
        uint32_t t[3][2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint32_t w = i < 4 ? x[(i + k) & 3] : y[(i + k) & 3];
            const uint32_t hi = w & 0xffff0000u;
            const float rest = __builtin_bit_cast(float, w) - __builtin_bit_cast(float, hi);
            const uint32_t mid = __builtin_bit_cast(uint32_t, rest) & 0xffff0000u;
            t[0][k] = hi;
            t[1][k] = mid;
            t[2][k] = __builtin_bit_cast(uint32_t, rest - __builtin_bit_cast(float, mid));
        }
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            const uint32_t pair = __builtin_amdgcn_perm(t[n][1], t[n][0], 0x07060302);
            const phx_u2 both = {pair, 0};
            r.v[n][i] = __builtin_bit_cast(__bf16, (uint16_t)both.x);
            r.v[n][i + 1] = __builtin_bit_cast(__bf16, (uint16_t)(both.x >> 16));
        }
    }
}

// Eight codes less their zero point, exactly.
__device__ __forceinline__ phx_h8 codes(uint32_t w, int zero, uint32_t one, _Float16) {
    const uint32_t mask = 0x000f000f;
    const phx_u4 x = {(w & mask) | one, (w >> 4 & mask) | one, (w >> 8 & mask) | one,
                      (w >> 12 & mask) | one};  // 1024 + code
    const _Float16 z = __builtin_bit_cast(_Float16, (uint16_t)(0x6400 + zero));
    return __builtin_bit_cast(phx_h8, x) - (phx_h8){z, z, z, z, z, z, z, z};
}
__device__ __forceinline__ b8 codes(uint32_t w, int zero, uint32_t, float) {
    const float z = (float)zero;
    const uint32_t lo = w & 0x0f0f0f0f, hi = w >> 4 & 0x0f0f0f0f;
    phx_u4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // elements 2i and 2i + 1: nibbles i and i + 4
        const uint32_t src = i & 1 ? hi : lo;
        const float a = (float)(src >> (8 * (i / 2)) & 255) - z;
        const float b = (float)(src >> (8 * (i / 2 + 2)) & 255) - z;
        x[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a),
                                     0x07060302);
    }
    return __builtin_bit_cast(b8, x);
}

__device__ __forceinline__ phx_f4 product(const Rows<_Float16> &a, phx_h8 w, phx_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v, w, c, 0, 0, 0);
}
__device__ __forceinline__ phx_f4 product(const Rows<float> &a, b8 w, phx_f4 c) {
    // the small terms first
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[2], w, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[1], w, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[0], w, c, 0, 0, 0);
}

// A workgroup: NT tiles of 16 columns, MT tiles of 16 rows, its waves over the
// tiles of K in turns; they add up in LDS.  PER groups in a tile.
template <typename T, int MT, int NT, int WAVES, int PER>
__device__ __forceinline__ void gemv_w4(const PhxGemvW4 &p) {
    __shared__ phx_f4 part[WAVES * MT * NT * 64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t r = lane & 15, quad = lane >> 4;
    const int64_t kb = (p.K + 127) / 128, n0 = (int64_t)blockIdx.x * (16 * NT);
    const uint32_t one = in_vgpr(0x64006400);
    const __amdgpu_buffer_rsrc_t a = __builtin_amdgcn_make_buffer_rsrc(
        (void *)p.a, 0, (int)(((p.M - 1) * p.lda + p.K) * sizeof(T)), 0x00020000);
    phx_f4 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[n][m] = (phx_f4){0, 0, 0, 0};

    struct Block {
        phx_u4 w[NT];
        _Float16 s[NT][PER];
        int z[NT][PER];
    };
    auto fetch = [&](Block &t, int64_t b) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            // (columns past N read the last one's, and are not stored)
            int64_t col = n0 + 16 * n + r;
            if (col >= p.N) col = p.N - 1;
            t.w[n] = *(const PHX_GLOBAL phx_u4 *)((const PHX_GLOBAL char *)p.w +
                                                 ((col / 16 * kb + b) * 64 + quad * 16 + col % 16) * 16);
#pragma unroll
            for (int g = 0; g < PER; ++g) {
                int64_t group = b * PER + g;
                if (group >= p.groups) group = p.groups - 1;
                t.s[n][g] = ((const PHX_GLOBAL _Float16 *)p.scales)[group * p.N + col];
                t.z[n][g] = p.zeros ? ((const PHX_GLOBAL uint8_t *)p.zeros)[group * p.N + col] : 8;
            }
        }
    };
    auto multiply = [&](const Block &t, int64_t b) {
#pragma unroll
        for (int g = 0; g < PER; ++g) {
            phx_f4 sum[NT][MT];
#pragma unroll
            for (int j = g * (4 / PER); j < (g + 1) * (4 / PER); ++j) {
                const uint32_t k = (uint32_t)b * 128 + 32 * j + 8 * quad;
                Rows<T> x[MT];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const uint32_t row = 16 * m + r;
                    // past the resource's end: zeros
                    load(x[m], a, row < p.M && k < p.K ? (uint32_t)((row * p.lda + k) * sizeof(T))
                                                       : 0x80000000u);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const auto w = codes(t.w[n][j], t.z[n][g], one, T());
#pragma unroll
                    for (int m = 0; m < MT; ++m)
                        sum[n][m] = product(x[m], w, j == g * (4 / PER) ? (phx_f4){0, 0, 0, 0}
                                                                        : sum[n][m]);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[n][m][i] = fmaf((float)t.s[n][g], sum[n][m][i], acc[n][m][i]);
        }
    };
    Block t, t2;
    const int64_t first = __builtin_amdgcn_readfirstlane(wave);
    if (first < kb) fetch(t, first);
    if (first + WAVES < kb) fetch(t2, first + WAVES);
    for (int64_t b = first; b < kb; b += 2 * WAVES) {
        multiply(t, b);
        if (b + 2 * WAVES < kb) fetch(t, b + 2 * WAVES);
        if (b + WAVES < kb) multiply(t2, b + WAVES);
        if (b + 3 * WAVES < kb) fetch(t2, b + 3 * WAVES);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) part[((wave * NT + n) * MT + m) * 64 + lane] = acc[n][m];
    __syncthreads();
    // a lane's four sums: column r, rows 4 quad .. 4 quad + 3 of the tile
    for (uint32_t x = threadIdx.x; x < NT * MT * 64; x += 64 * WAVES) {
        phx_f4 sum = part[x];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) sum = sum + part[w * (NT * MT * 64) + x];
        const int64_t col = n0 + x / (MT * 64) * 16 + (x & 15);
        const uint32_t row = x / 64 % MT * 16 + (x >> 4 & 3) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (col < p.N && row + i < p.M) {
                PHX_GLOBAL T *c = (PHX_GLOBAL T *)p.c + (row + i) * p.ldc + col;
                float o = p.alpha * sum[i];
                if (p.beta != 0.0f) o = o + p.beta * (float)*c;
                *c = (T)o;
            }
    }
}

}  // namespace

#define GEMV(T, suffix, MT, NT, WAVES, PER)                                                     \
    extern "C" __global__ __launch_bounds__(64 * WAVES) void                                    \
        gemv_w4_##suffix##_m##MT##_n##NT##_g##PER(PhxGemvW4 p) {                                \
        gemv_w4<T, MT, NT, WAVES, PER>(p);                                                      \
    }
#define GROUPS(T, suffix, MT, NT, WAVES)                                                        \
    GEMV(T, suffix, MT, NT, WAVES, 1)                                                           \
    GEMV(T, suffix, MT, NT, WAVES, 2)                                                           \
    GEMV(T, suffix, MT, NT, WAVES, 4)
GROUPS(_Float16, f16, 1, 1, 8)
GROUPS(_Float16, f16, 2, 1, 8)
GROUPS(_Float16, f16, 4, 1, 8)
GROUPS(float, f32, 1, 1, 8)
GROUPS(float, f32, 2, 1, 8)
GROUPS(float, f32, 4, 1, 8)
