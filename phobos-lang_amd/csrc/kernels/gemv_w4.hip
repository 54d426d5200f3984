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
//
// Few rows are bound by the codes' bytes, and by latency where those are few:
// every code is read once, two blocks of a wave ahead. 16384 x 8192 in groups of
// 128, f16: 1 row 16.7 us (4.2 TB/s), 16 rows 19.4 us; f32: 27.1 and 35.9 us.
// 64 rows of 16384 x 8192 take 30.2 us (570 TFLOP/s; f32 60.8 us). Of a CU's cycles
// the vector instructions are busy 48 %, LDS 41 % (a row's operand read from
// it serves one product) and the matrix cores 26 %, which four waves a SIMD
// overlap in part.
// A split of N in tiles leaves CUs idle below 4096 columns; there 8 to 16 waves
// share a tile's K. A scale and a zero point are loaded by a quarter of a wave
// for the groups of a block and handed around by the lanes. Groups of 32 cost
// more than their bytes (zero points, 16384 x 8192, f16: 1 row 21.5 us against 16.6
// in groups of 128, 64 rows 40.1 against 31.8).
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

// Rows of A as matrix operands: of each k one f16 term, or three bf16 terms of an
// f32, which hold its 24 bits (those from 2^-126 up: the matrix instructions
// take a bf16 below its normal numbers as 0).
template <typename T>
struct Rows;
template <>
struct Rows<_Float16> {
    static constexpr int TERMS = 1;
    phx_h8 v[1];
};
template <>
struct Rows<float> {
    static constexpr int TERMS = 3;
    b8 v[3];
};

// 16 rows of a block of 128 k go through LDS: in memory a lane's neighbours have
// the next k of the same row (a wave's load of 16 rows by 64 bytes, as the
// operands have them, takes 64 cycles of the CU's vector memory path, one a
// lane, where whole rows take 16), in the operands the same k of the next.
// A term's 16 bytes of row r and k 8c .. 8c+7 are at 256 c + 16 (r ^ c): writes
// and reads of 16 lanes touch every bank once.
constexpr uint32_t kTile = 4096;  // bytes of 16 rows of one term

template <typename T>
struct Staged {
    static constexpr uint32_t ROWS = sizeof(T) == 2 ? 4 : 2;  // of a wave's load
    static constexpr uint32_t LOADS = 16 / ROWS;              // for 16 rows
    static constexpr uint32_t BYTES = kTile * Rows<T>::TERMS;

    // the lane's row and first k in a block in load f of its rows
    static __device__ __forceinline__ uint32_t row(uint32_t f, uint32_t lane) {
        return f * ROWS + lane / (64 / ROWS);
    }
    static __device__ __forceinline__ uint32_t k(uint32_t lane) {
        return lane % (64 / ROWS) * (16 / sizeof(T));
    }
    static __device__ __forceinline__ uint32_t at(uint32_t row, uint32_t c) {
        return c * 256 + ((row ^ c) & 15) * 16;
    }
    // `lds`: the 16 rows' part
    static __device__ __forceinline__ void put(char *lds, phx_u4 x, uint32_t row, uint32_t lane) {
        if constexpr (sizeof(T) == 2) {
            *(phx_u4 *)(lds + at(row, lane % 16)) = x;
        } else {
            phx_u2 out[3];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // the top 16 bits, what they leave, and what that leaves: each exact
                uint32_t t[3][2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t w = x[2 * i + k], hi = w & 0xffff0000u;
                    const float rest = __builtin_bit_cast(float, w) - __builtin_bit_cast(float, hi);
                    const uint32_t mid = __builtin_bit_cast(uint32_t, rest) & 0xffff0000u;
                    t[0][k] = hi;
                    t[1][k] = mid;
                    t[2][k] = __builtin_bit_cast(uint32_t, rest - __builtin_bit_cast(float, mid));
                }
#pragma unroll
                for (int n = 0; n < 3; ++n)
                    out[n][i] = __builtin_amdgcn_perm(t[n][1], t[n][0], 0x07060302);
            }
#pragma unroll
            for (int n = 0; n < 3; ++n)
                *(phx_u2 *)(lds + n * kTile + at(row, lane % 32 / 2) + lane % 2 * 8) = out[n];
        }
    }
    // the operand of the block's j-th 32 k
    static __device__ __forceinline__ Rows<T> get(const char *lds, int j, uint32_t lane) {
        Rows<T> r;
#pragma unroll
        for (int n = 0; n < Rows<T>::TERMS; ++n)
            r.v[n] = __builtin_bit_cast(
                __typeof__(r.v[n]), *(const phx_u4 *)(lds + n * kTile + at(lane & 15, 4 * j + lane / 16)));
        return r;
    }
};

// Eight codes less their zero point, exactly.
__device__ __forceinline__ phx_h8 codes(uint32_t w, int zero, const uint32_t (&one)[2], _Float16) {
    const uint32_t low = 0x000f000f, high = 0x00f000f0;
    // 1024 + code in the low nibbles of a half's byte, 64 + code in the high
    const _Float16 z = (_Float16)(1024 + zero), y = (_Float16)(64 + zero);
    const phx_h2 zz = {z, z}, yy = {y, y};
    auto less = [](uint32_t x, phx_h2 y) {
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(phx_h2, x) - y);
    };
    const uint32_t v = w >> 8;
    const phx_u4 x = {less((w & low) | one[0], zz), less((w & high) | one[1], yy),
                      less((v & low) | one[0], zz), less((v & high) | one[1], yy)};
    return __builtin_bit_cast(phx_h8, x);
}
__device__ __forceinline__ b8 codes(uint32_t w, int zero, const uint32_t (&)[2], float) {
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
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[0], w, c, 0, 0, 0);
}
__device__ __forceinline__ phx_f4 product(const Rows<float> &a, b8 w, phx_f4 c) {
    // the small terms first
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[2], w, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[1], w, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[0], w, c, 0, 0, 0);
}

// The weights of a 128-row block of NT tiles of columns, as loaded: of its PER
// groups a lane has the scale and the zero point of the (lane / 16 % PER)-th.
template <int NT>
struct Block {
    phx_u4 w[NT];
    uint16_t s[NT];
    uint8_t z[NT];
};

// A lane's columns, 16 n + lane % 16 from n0 on, in the codes and the groups.
// Addresses are a scalar base and a lane's 32-bit offset.
template <int NT, int PER>
struct Columns {
    uint32_t col[NT], lane_w, group;
    int64_t tile[NT];  // its first block

    __device__ __forceinline__ void start(const PhxGemvW4 &p, int64_t n0, int64_t kb, uint32_t lane) {
        lane_w = (lane >> 4) * 256 + (lane & 15) * 16;
        group = lane / 16 % PER;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            // columns past N read the last one's, and tiles past it the last
            // one, and are not stored
            const int64_t c = n0 + 16 * n + (lane & 15), last = (p.N - 1) / 16;
            col[n] = (uint32_t)(c < p.N ? c : p.N - 1);
            tile[n] = (n0 / 16 + n < last ? n0 / 16 + n : last) * kb;
        }
    }
    __device__ __forceinline__ void fetch(const PhxGemvW4 &p, Block<NT> &t, uint32_t b) const {
#pragma unroll
        for (int n = 0; n < NT; ++n)
            t.w[n] = *(const PHX_GLOBAL phx_u4 *)((const PHX_GLOBAL char *)p.w +
                                                  (tile[n] + b) * 1024 + lane_w);
        const int64_t first = (int64_t)b * PER * p.N;
        const uint32_t left = (uint32_t)p.groups - 1 - b * PER;  // groups behind the first
        const uint32_t at = (PER == 1 ? 0 : min(group, left)) * (uint32_t)p.N;
        const PHX_GLOBAL uint16_t *s = (const PHX_GLOBAL uint16_t *)p.scales + first;
        const PHX_GLOBAL uint8_t *z = (const PHX_GLOBAL uint8_t *)p.zeros + first;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            t.s[n] = s[at + col[n]];
            t.z[n] = p.zeros ? z[at + col[n]] : 8;
        }
    }
};

// The j-th 32 rows of a block: its products, and at the end of a group their
// sum, scaled.
template <typename T, int MT, int NT, int PER>
__device__ __forceinline__ void step(const Block<NT> &t, const Rows<T> (&rows)[MT], int j,
                                     uint32_t lane, const uint32_t (&one)[2],
                                     uint32_t (&group)[NT], phx_f4 (&sum)[NT][MT],
                                     phx_f4 (&acc)[NT][MT]) {
    constexpr int EACH = 4 / PER;  // of a group
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (j % EACH == 0) {
            group[n] = (uint32_t)t.z[n] << 16 | t.s[n];
            if (PER > 1)
                group[n] = __builtin_amdgcn_ds_bpermute(
                    (int)((lane & 15) + 16 * (j / EACH)) * 4, (int)group[n]);
        }
        const auto w = codes(t.w[n][j], (int)(group[n] >> 16), one, T());
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            sum[n][m] = product(rows[m], w, j % EACH ? sum[n][m] : (phx_f4){0, 0, 0, 0});
            if (j % EACH == EACH - 1) {
                const float s = (float)__builtin_bit_cast(_Float16, (uint16_t)group[n]);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[n][m][i] = fmaf(s, sum[n][m][i], acc[n][m][i]);
            }
        }
    }
}

// Stores a lane's four sums: column c, rows row .. row + 3; to C, or a part of a
// split as it is.
template <typename T>
__device__ __forceinline__ void store(const PhxGemvW4 &p, phx_f4 sum, int64_t c, uint32_t row) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (c < p.N && row + i < p.M) {
            if (p.splits > 1) {
                ((PHX_GLOBAL float *)p.ws)[((int64_t)blockIdx.z * p.M + row + i) * p.N + c] = sum[i];
                continue;
            }
            PHX_GLOBAL T *to = (PHX_GLOBAL T *)p.c + (row + i) * p.ldc + c;
            float o = p.alpha * sum[i];
            if (p.beta != 0.0f) o = o + p.beta * (float)*to;
            *to = (T)o;
        }
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const PhxGemvW4 &p, size_t size) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)p.a, 0,
                                             (int)(((p.M - 1) * p.lda + p.K) * size), 0x00020000);
}

// 16 rows: a workgroup takes NT tiles of 16 columns, its waves the blocks of K in
// turns, each with the rows it needs in its own part of LDS; they add up
// at the end.
template <typename T, int NT, int WAVES, int PER>
__device__ __forceinline__ void gemv_w4(const PhxGemvW4 &p) {
    using St = Staged<T>;
    __shared__ phx_u4 lds[WAVES * St::BYTES / 16];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t kb = (p.K + 127) / 128, n0 = (int64_t)blockIdx.x * (16 * NT);
    const uint32_t one[2] = {in_vgpr(0x64006400), in_vgpr(0x54005400)};
    const __amdgpu_buffer_rsrc_t a = rows_of(p, sizeof(T));
    char *own = (char *)lds + wave * St::BYTES;
    phx_f4 acc[NT][1];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = (phx_f4){0, 0, 0, 0};
    Columns<NT, PER> columns;
    columns.start(p, n0, kb, lane);
    // rows and k that do not exist lie past the resource's end: zeros; loads of
    // none but such rows are left out, and their part of LDS keeps its zeros
    const uint32_t m0 = blockIdx.y * 16;
    const uint32_t loads = (min((uint32_t)p.M - m0, 16u) + St::ROWS - 1) / St::ROWS;
    struct Share {
        phx_u4 x[St::LOADS];
    };
    auto fetch = [&](Share &x, Block<NT> &t, uint32_t b) {
        const uint32_t k = b * 128 + St::k(lane);
#pragma unroll
        for (uint32_t f = 0; f < St::LOADS; ++f)
            if (f < loads) {
                const uint32_t row = m0 + St::row(f, lane);
                x.x[f] = __builtin_amdgcn_raw_buffer_load_b128(
                    a, row < p.M && k < p.K ? (uint32_t)((row * p.lda + k) * sizeof(T)) : 0x80000000u,
                    0, 0);
            }
        columns.fetch(p, t, b);
    };
    auto multiply = [&](const Share &x, const Block<NT> &t) {
#pragma unroll
        for (uint32_t f = 0; f < St::LOADS; ++f)
            if (f < loads) St::put(own, x.x[f], St::row(f, lane), lane);
        uint32_t group[NT];
        phx_f4 sum[NT][1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const Rows<T> rows[1] = {St::get(own, j, lane)};
            step<T, 1, NT, PER>(t, rows, j, lane, one, group, sum, acc);
        }
    };
    Share x, x2;
    Block<NT> t, t2;
    const uint32_t first = __builtin_amdgcn_readfirstlane(wave), end = (uint32_t)kb;
    if (first < end) fetch(x, t, first);
    if (first + WAVES < end) fetch(x2, t2, first + WAVES);
    for (uint32_t i = lane; i < St::BYTES / 16; i += 64) ((phx_u4 *)own)[i] = (phx_u4){0, 0, 0, 0};
    for (uint32_t b = first; b < end; b += 2 * WAVES) {
        multiply(x, t);
        if (b + 2 * WAVES < end) fetch(x, t, b + 2 * WAVES);
        if (b + WAVES < end) multiply(x2, t2);
        if (b + 3 * WAVES < end) fetch(x2, t2, b + 3 * WAVES);
    }
    // a lane's four sums: column lane % 16, rows 4 (lane / 16) .. + 3
    phx_f4 *part = (phx_f4 *)lds;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        __syncthreads();
        part[wave * 64 + lane] = acc[n][0];
        __syncthreads();
        if (wave) continue;
        phx_f4 sum = part[lane];
#pragma unroll
        for (int v = 1; v < WAVES; ++v) sum = sum + part[v * 64 + lane];
        store<T>(p, sum, n0 + 16 * n + (lane & 15), m0 + lane / 16 * 4);
    }
}

// More rows: a workgroup takes WN tiles of columns and MT of rows, and its WN x WK
// waves share the rows through LDS: WK blocks of K at a time, split into their
// matrix terms once, each read by the WN waves of a block.  (16 waves with a tile
// of columns each: 64 x 16384 x 8192 f16 30.2 us, with 8 waves of two 36.5 and of
// four rows' tiles as well 33.8, however far ahead they load.)
// One barrier for every WK blocks: the next ones are loaded into registers
// while these are multiplied, and written to the other half of LDS.
template <typename T, int MT, int WN, int WK, int PER>
__device__ __forceinline__ void gemm_w4(const PhxGemvW4 &p) {
    using St = Staged<T>;
    constexpr uint32_t EACH = MT * St::LOADS / WN;       // a wave's loads of its block
    constexpr uint32_t STAGE = WK * MT * St::BYTES;
    constexpr uint32_t SUMS = WK * WN * MT * 1024;
    __shared__ phx_u4 lds[(2 * STAGE > SUMS ? 2 * STAGE : SUMS) / 16];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t wn = __builtin_amdgcn_readfirstlane(wave % WN);
    const uint32_t wk = __builtin_amdgcn_readfirstlane(wave / WN);
    const int64_t kb = (p.K + 127) / 128, n0 = ((int64_t)blockIdx.x * WN + wn) * 16;
    const uint32_t m0 = blockIdx.y * (16 * MT);
    const uint32_t per = ((uint32_t)kb + p.splits - 1) / p.splits;
    const uint32_t begin = blockIdx.z * per, end = min(begin + per, (uint32_t)kb);
    const uint32_t one[2] = {in_vgpr(0x64006400), in_vgpr(0x54005400)};
    const __amdgpu_buffer_rsrc_t a = rows_of(p, sizeof(T));
    Columns<1, PER> columns;
    columns.start(p, n0, kb, lane);
    phx_u4 x[EACH];
    // a wave with no block left multiplies zero rows with the last block's codes
    auto fetch = [&](Block<1> &t, uint32_t b) {
        const uint32_t k = b * 128 + St::k(lane);
#pragma unroll
        for (uint32_t e = 0; e < EACH; ++e) {
            const uint32_t row = m0 + St::row(wn * EACH + e, lane);
            x[e] = __builtin_amdgcn_raw_buffer_load_b128(
                a, row < p.M && k < p.K && b < end ? (uint32_t)((row * p.lda + k) * sizeof(T))
                                                   : 0x80000000u, 0, 0);
        }
        columns.fetch(p, t, min(b, (uint32_t)kb - 1));
    };
    phx_f4 acc[1][MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[0][m] = (phx_f4){0, 0, 0, 0};
    Block<1> t, next;
    fetch(next, begin + wk);
    for (uint32_t b = begin, half = 0; b < end; b += WK, half ^= 1) {
        char *block = (char *)lds + half * STAGE + wk * (MT * St::BYTES);
        t = next;
#pragma unroll
        for (uint32_t e = 0; e < EACH; ++e) {
            const uint32_t row = St::row(wn * EACH + e, lane);
            St::put(block + row / 16 * St::BYTES, x[e], row, lane);
        }
        __syncthreads();
        if (b + WK < end) fetch(next, b + WK + wk);
        uint32_t group[1];
        phx_f4 sum[1][MT];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            Rows<T> rows[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) rows[m] = St::get(block + m * St::BYTES, j, lane);
            step<T, MT, 1, PER>(t, rows, j, lane, one, group, sum, acc);
        }
    }
    __syncthreads();
    phx_f4 *part = (phx_f4 *)lds;
#pragma unroll
    for (int m = 0; m < MT; ++m) part[((wk * WN + wn) * MT + m) * 64 + lane] = acc[0][m];
    __syncthreads();
    constexpr uint32_t EVERY = WN * MT * 64;
    for (uint32_t i = threadIdx.x; i < EVERY; i += 64 * WN * WK) {
        phx_f4 sum = part[i];
#pragma unroll
        for (int v = 1; v < WK; ++v) sum = sum + part[v * EVERY + i];
        const uint32_t m = i / 64 % MT, tile = i / (64 * MT);
        store<T>(p, sum, ((int64_t)blockIdx.x * WN + tile) * 16 + (i & 15),
                 m0 + 16 * m + (i >> 4 & 3) * 4);
    }
}

}  // namespace

#define GEMV(T, suffix, NT, WAVES, PER)                                                         \
    extern "C" __global__ __launch_bounds__(64 * WAVES) void                                    \
        gemv_w4_##suffix##_n##NT##_w##WAVES##_g##PER(PhxGemvW4 p) {                             \
        gemv_w4<T, NT, WAVES, PER>(p);                                                          \
    }
#define GROUPS(T, suffix, NT, WAVES)                                                            \
    GEMV(T, suffix, NT, WAVES, 1)                                                               \
    GEMV(T, suffix, NT, WAVES, 2)                                                               \
    GEMV(T, suffix, NT, WAVES, 4)
#define GEMM(T, suffix, MT, WN, WK, PER)                                                        \
    extern "C" __global__ __launch_bounds__(64 * WN * WK) void                                  \
        gemm_w4_##suffix##_m##MT##_##WN##x##WK##_g##PER(PhxGemvW4 p) {                          \
        gemm_w4<T, MT, WN, WK, PER>(p);                                                         \
    }
#define GEMM_GROUPS(T, suffix, MT, WN, WK)                                                      \
    GEMM(T, suffix, MT, WN, WK, 1)                                                              \
    GEMM(T, suffix, MT, WN, WK, 2)                                                              \
    GEMM(T, suffix, MT, WN, WK, 4)
// (Three f32 forms spill registers: n2_w12 in groups of 64 and 32 8 and 42 of 168,
// n4_w8 in groups of 32 32 of 256.  16 rows in groups of 128, 64 and 32: 8192 x 4096
// in the first 13.5, 14.5 and 19.1 us, 16384 x 8192 in the second 35.7, 36.9 and 45.6;
// 1 row 26.8, 27.7 and 29.3.)
GROUPS(_Float16, f16, 1, 8)
GROUPS(_Float16, f16, 1, 16)
GROUPS(_Float16, f16, 4, 8)
GROUPS(float, f32, 1, 12)
GROUPS(float, f32, 2, 12)
GROUPS(float, f32, 4, 8)
GEMM_GROUPS(_Float16, f16, 4, 4, 4)
GEMM_GROUPS(_Float16, f16, 2, 4, 4)
GEMM_GROUPS(_Float16, f16, 2, 2, 8)
GEMM_GROUPS(float, f32, 4, 16, 1)
GEMM_GROUPS(float, f32, 2, 8, 2)
GEMM_GROUPS(float, f32, 2, 4, 2)

// C from the parts of a split, in order.
template <typename T>
__device__ __forceinline__ void reduce(const PhxGemvW4 &p) {
    const int64_t plane = p.M * p.N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < plane;
         i += (int64_t)gridDim.x * 256) {
        const PHX_GLOBAL float *part = (const PHX_GLOBAL float *)p.ws + i;
        float sum = part[0];
        for (int v = 1; v < p.splits; ++v) sum += part[v * plane];
        PHX_GLOBAL T *to = (PHX_GLOBAL T *)p.c + i / p.N * p.ldc + i % p.N;
        float o = p.alpha * sum;
        if (p.beta != 0.0f) o = o + p.beta * (float)*to;
        *to = (T)o;
    }
}
extern "C" __global__ __launch_bounds__(256) void gemm_w4_reduce_f16(PhxGemvW4 p) {
    reduce<_Float16>(p);
}
extern "C" __global__ __launch_bounds__(256) void gemm_w4_reduce_f32(PhxGemvW4 p) {
    reduce<float>(p);
}
