// Kernels that write rows in 8 bits: the root-mean-square norm with the
// residual's addition, and the gated activation (the layout and the arithmetic:
// include/phobos_hip.h, phx_norm_f8 and phx_glu_f8).
#include "f8.h"

namespace {

template <typename T>
struct Chunk {  // 16 bytes of a row
    static constexpr int N = 16 / sizeof(T);
    static constexpr int LANES = PHX_F8_BLOCK / N;  // of a scale's block
    float v[N];

    __device__ __forceinline__ void load(const PHX_GLOBAL T *p) { of(*(const PHX_GLOBAL phx_u4 *)p); }
    __device__ __forceinline__ void of(phx_u4 w) {
        if constexpr (sizeof(T) == 2) {
            const phx_h8 h = __builtin_bit_cast(phx_h8, w);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = (float)h[i];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = __builtin_bit_cast(float, (uint32_t)w[i]);
        }
    }
    __device__ __forceinline__ void store(PHX_GLOBAL T *p) const {
        if constexpr (sizeof(T) == 2) {
            phx_h8 h;
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] = (_Float16)v[i];
            *(PHX_GLOBAL phx_h8 *)p = h;
        } else {
            *(PHX_GLOBAL phx_f4 *)p = (phx_f4){v[0], v[1], v[2], v[3]};
        }
    }
};

// The largest magnitude of a block, in all its lanes (of a row's `lanes`, if they are fewer).
template <int LANES>
__device__ __forceinline__ uint32_t block_largest(uint32_t a, uint32_t lanes = LANES) {
#pragma unroll
    for (uint32_t s = 1; s < LANES; s <<= 1)
        if (s < lanes) a = max(a, (uint32_t)__shfl_xor((int)a, (int)s));
    return a;
}

template <typename T>
__device__ __forceinline__ void store_codes(const PhxF8Rows &p, int64_t row, uint32_t k,
                                            const float (&t)[Chunk<T>::N], uint32_t a) {
    uint32_t out[Chunk<T>::N / 4];
    f8_codes(t, a, out);
    PHX_GLOBAL char *to = (PHX_GLOBAL char *)p.q + row * p.ldq + k;
    if constexpr (sizeof(T) == 2)
        *(PHX_GLOBAL phx_u2 *)to = (phx_u2){out[0], out[1]};
    else
        *(PHX_GLOBAL uint32_t *)to = out[0];
}

// The threads that a row is given: a workgroup, or (ROWS) a wave or the 2, 4 .. 32 lanes that
// its chunks take.
template <typename T, int C, bool ROWS>
__device__ __forceinline__ uint32_t threads_of_row(uint32_t K) {
    if (!ROWS) return blockDim.x;
    const uint32_t chunks = K / Chunk<T>::N;
    return C > 1 || chunks > 32 ? 64 : 1u << (32 - __builtin_clz(chunks - 1));
}

// Threads next to each other take a row, chunks of 16 bytes next to their neighbours', up
// to C chunks a thread, which stay in registers between the sum and what follows it: every
// byte is read once and written once.
// Long runs are bound by memory: 16384 rows of 8192, f16, with the sum, 162-166 us
// (5.8 TB/s; a copy, which writes as much as it reads, 5.1), the vector instructions
// busy two thirds of it (the squares in 64 bits, the codes' exact quotients). Fewer
// rows than the GPU holds at once are one chain of load, sum, divide and store: 1000
// of 4144, f32, 9.3 us, one of 4096, f16, 3.0. A row per workgroup rather than several
// turns of a wave: a second reading would come from memory. (Two chunks a thread, not
// four or one, where there are many rows: the figures are with the rule that chooses.)
template <typename T, int C, bool ROWS>
__device__ __forceinline__ void norm_f8(const PhxF8Rows &p) {
    constexpr int N = Chunk<T>::N;
    __shared__ double sums[16];
    const uint32_t K = (uint32_t)p.K, R = threads_of_row<T, C, ROWS>(K), waves = R / 64;
    const int64_t row = ROWS ? (int64_t)blockIdx.x * (256 / R) + threadIdx.x / R : (int64_t)blockIdx.x;
    const uint32_t at = (ROWS ? threadIdx.x % R : threadIdx.x) * N;
    if (ROWS && row >= p.M) return;  // (lanes of another row need none of it)
    Chunk<T> h[C];
    // (asked for with the rows: it is in use as soon as their sum is there; of eight chunks a
    // thread, for all of which there are no registers, one ahead)
    constexpr int EARLY = C == 8 ? 1 : C;
    phx_u4 gain[C];
    auto load_gain = [&](int c, uint32_t k) {
        gain[c] = *(const PHX_GLOBAL phx_u4 *)((const PHX_GLOBAL T *)p.gain + k);
    };
    double sum = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t k = at + c * (R * N);
#pragma unroll
        for (int i = 0; i < N; ++i) h[c].v[i] = 0;
        if (k >= K) continue;
        if (c < EARLY) load_gain(c, k);
        h[c].load((const PHX_GLOBAL T *)p.x + row * p.ldx + k);
        if (p.r) {
            Chunk<T> r;
            r.load((const PHX_GLOBAL T *)p.r + row * p.ldr + k);
            // what is stored is what the norm reads
#pragma unroll
            for (int i = 0; i < N; ++i) h[c].v[i] = (float)(T)(h[c].v[i] + r.v[i]);
        }
        if (p.h) h[c].store((PHX_GLOBAL T *)p.h + row * p.ldh + k);
        // squares of f32 are exact in 64 bits and leave its range nowhere
#pragma unroll
        for (int i = 0; i < N; ++i) sum = fma((double)h[c].v[i], (double)h[c].v[i], sum);
    }
#pragma unroll
    for (uint32_t s = 1; s < 64; s <<= 1)
        if (!ROWS || s < R) sum += __shfl_xor(sum, (int)s);
    if (!ROWS && waves > 1) {
        if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
        __syncthreads();
        sum = sums[0];
        for (uint32_t w = 1; w < waves; ++w) sum += sums[w];
    }
    const double factor = rsqrt(sum * p.inverse + (double)p.eps);
    const float f = (float)factor;
    // (rows of the smallest or largest f32, where f has few bits or none)
    const bool plain = f >= 0x1p-126f && f <= 0x1.fp127f;
    const bool all_plain = ROWS ? __all(plain) : __builtin_amdgcn_readfirstlane(plain);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t k = at + c * (R * N);
        const bool live = k < K;
        uint32_t a = 0;
        if (EARLY < C) {
            if (c + 1 < C && k + R * N < K) load_gain(c + 1, k + R * N);
            // (else the chunks are worked on together, in more registers than there are)
            __builtin_amdgcn_sched_barrier(0);
        }
        if (live) {
            Chunk<T> g;
            g.of(gain[c]);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                h[c].v[i] = h[c].v[i] * g.v[i];
                a = max(a, f8_magnitude(h[c].v[i]));
            }
        }
        if (p.q) {
            a = block_largest<Chunk<T>::LANES>(a, ROWS ? R : 64);
            if (live) {
                store_codes<T>(p, row, k, h[c].v, a);
                if (at % PHX_F8_BLOCK == 0)
                    ((PHX_GLOBAL float *)p.scales)[row * p.lds + k / PHX_F8_BLOCK] =
                        a < 0x7f800000u
                            ? (float)((double)__builtin_bit_cast(float, a) * (factor * (1 / 448.0)))
                            : __builtin_nanf("");
            }
        }
        if (p.y && live) {
            if (all_plain) {
#pragma unroll
                for (int i = 0; i < N; ++i) h[c].v[i] *= f;
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    h[c].v[i] = plain ? h[c].v[i] * f : (float)((double)h[c].v[i] * factor);
            }
            h[c].store((PHX_GLOBAL T *)p.y + row * p.ldy + k);
        }
    }
}

// x log2(e) in two terms, so that a large x keeps its bits.
struct Power {
    float high, low;
    __device__ __forceinline__ explicit Power(float x) {
        const float e = 1.44269504f, rest = 1.92596303e-8f;  // log2(e) in two terms
        high = x * e;
        low = __builtin_fmaf(x, rest, __builtin_fmaf(x, e, -high));
    }
};

// e^x for x up to 80; below -100, where one plus it is one, that of -100.
__device__ __forceinline__ float exp_of(float x) {
    const Power p(fmaxf(x, -100.0f));
    const float y = __builtin_amdgcn_exp2f(p.high);
    return __builtin_fmaf(y * p.low, 0.693147181f, y);
}

// gate * e^gate * value: the activation of gates below -80, where 1 + e^gate is 1. From
// -88.7 on e^-gate is no f32 any more, and e^gate not one of all its bits, but their product
// with a large value is: the power of two is taken in halves, before and behind the product.
// (Where the first half leaves bits or all of the value below 2^-126, the result is 0.)
__device__ __forceinline__ float far_value(float gate, float value) {
    const float x = fmaxf(gate, -400.0f);  // (e^-400 times any two values is 0)
    const Power p(x);
    const float whole = rintf(p.high);
    const float e = __builtin_amdgcn_exp2f((p.high - whole) + p.low);
    const int n = (int)whole, half = n / 2;
    const float t = ldexpf(x * e * ldexpf(value, half), n - half);
    return gate == -INFINITY ? __builtin_nanf("") : t;
}

// A block of 128 of a row to 16 or 32 lanes; blocks of a row next to each other. No
// lane needs more than its own block's, so a launch is as wide as its data. Bound by
// memory: 4133 rows of 5520, f32, 38.9 us (5.3 TB/s; with a division of f32 for every
// value 43); 16384 of 8192, f16, 143 us (4.7 TB/s; 174), f32 204 (5.9 TB/s); 32 of 4096,
// f16, 3.7 us, one chain of load and store. Blocks of fewer than 128 leave lanes idle:
// 1562500 rows of 64, f16, 186 us (2.7 TB/s).
template <typename T>
__device__ __forceinline__ void glu_f8(const PhxF8Rows &p) {
    constexpr int N = Chunk<T>::N, LANES = Chunk<T>::LANES;
    const uint32_t blocks = ((uint32_t)p.K + PHX_F8_BLOCK - 1) / PHX_F8_BLOCK;
    const int64_t unit = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const int64_t row = unit / blocks;
    const uint32_t block = (uint32_t)(unit % blocks);
    const uint32_t k = block * PHX_F8_BLOCK + threadIdx.x % LANES * N;
    const bool live = row < p.M && k < p.K;
    Chunk<T> u, v;
    uint32_t a = 0;
    if (live) {
        const PHX_GLOBAL T *x = (const PHX_GLOBAL T *)p.x + row * p.ldx + k;
        u.load(x);
        v.load(x + p.K);
        float t[N];
        uint32_t far = 0, least = ~0u;  // of the gates' bits, their magnitudes
#pragma unroll
        for (int i = 0; i < N; ++i) {
            far = max(far, __builtin_bit_cast(uint32_t, u.v[i]));
            if (sizeof(T) == 4) least = min(least, f8_magnitude(u.v[i]));
            // (the reciprocal within 2^-23 of itself, as long as it is no denormal)
            t[i] = u.v[i] * __builtin_amdgcn_rcpf(1.0f + exp_of(-u.v[i])) * v.v[i];
        }
        // Gates below -80; f32 ones below 2^-124, of which half may not have its bits.
        if (far > __builtin_bit_cast(uint32_t, -80.0f) || least < 3u << 23) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (u.v[i] < -80.0f) t[i] = far_value(u.v[i], v.v[i]);
                if (sizeof(T) == 4 && fabsf(u.v[i]) < 0x1p-124f)
                    t[i] = (u.v[i] * 0x1p24f) * (v.v[i] * 0x1p-25f);
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            u.v[i] = t[i];
            a = max(a, f8_magnitude(t[i]));
        }
    }
    a = block_largest<LANES>(a);
    if (!live) return;
    store_codes<T>(p, row, k, u.v, a);
    if (threadIdx.x % LANES == 0)
        ((PHX_GLOBAL float *)p.scales)[row * p.lds + block] =
            a < 0x7f800000u ? __builtin_bit_cast(float, a) / 448.0f : __builtin_nanf("");
}

}  // namespace

#define NORM(T, suffix, C)                                                                      \
    extern "C" __global__ __launch_bounds__(1024) void norm_f8_##suffix##_c##C(PhxF8Rows p) {   \
        norm_f8<T, C, false>(p);                                                                \
    }
#define ROWS(T, suffix, C)                                                                      \
    extern "C" __global__ __launch_bounds__(256) void norm_f8_rows_##suffix##_c##C(PhxF8Rows p) { \
        norm_f8<T, C, true>(p);                                                                 \
    }
#define NORMS(T, suffix)                                                                        \
    ROWS(T, suffix, 1) ROWS(T, suffix, 2) NORM(T, suffix, 1) NORM(T, suffix, 2) NORM(T, suffix, 4)
NORMS(_Float16, f16)
NORMS(float, f32)
NORM(float, f32, 8)
extern "C" __global__ __launch_bounds__(256) void glu_f8_f16(PhxF8Rows p) { glu_f8<_Float16>(p); }
extern "C" __global__ __launch_bounds__(256) void glu_f8_f32(PhxF8Rows p) { glu_f8<float>(p); }
