// C = alpha*A@W + beta*C for up to 64 rows of A and 4-bit weights W with a
// scale and a zero point per group of K (the layout and the arithmetic:
// include/phobos_hip.h, phx_gemv_w4).
//
//   acc[m,n] = sum over groups g of s[g,n] * sum over k in g of a[m,k] (q[k,n] - z[g,n])
//
// The inner sum is in f32 of exact products, scaled in f32.
#include "phx_common.h"
#include "phx_decode.h"

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

template <typename T>
__device__ __forceinline__ void gemv_w4(const PhxGemvW4 &p) {
    // a wave per output column and row of A, its lanes over the dwords of K
    const int lane = threadIdx.x & 63;
    const int64_t n = (int64_t)blockIdx.x * 4 + threadIdx.x / 64, m = blockIdx.y;
    if (n >= p.N) return;
    const int64_t kb = (p.K + 127) / 128;
    const uint32_t *w = (const uint32_t *)p.w + n / 16 * kb * 256;
    const _Float16 *scales = (const _Float16 *)p.scales;
    const uint8_t *zeros = (const uint8_t *)p.zeros;
    const T *a = (const T *)p.a + m * p.lda;
    float acc = 0.0f;
    for (int64_t d = lane; d * 8 < p.K; d += 64) {  // k = 8 d .. 8 d + 7
        const int64_t b = d / 16;
        const int j = (int)(d % 16) / 4, q = d % 4;
        const uint32_t word = w[b * 256 + (q * 16 + n % 16) * 4 + j];
        const int64_t g = d * 8 / p.group * p.N + n;
        const int z = zeros ? zeros[g] : 8;
        float part = 0.0f;
        for (int e = 0; e < 8; ++e) {
            const int c = (word >> (4 * (e / 2 + 4 * (e % 2)))) & 15;
            part = fmaf((float)a[d * 8 + e], (float)(c - z), part);
        }
        acc = fmaf((float)scales[g], part, acc);
    }
    for (int s = 32; s; s >>= 1) acc += __shfl_xor(acc, s);
    if (lane == 0) {
        T *c = (T *)p.c + m * p.ldc + n;
        float o = p.alpha * acc;
        if (p.beta != 0.0f) o = o + p.beta * (float)*c;
        *c = (T)o;
    }
}

extern "C" __global__ __launch_bounds__(256) void gemv_w4_f16(PhxGemvW4 p) {
    gemv_w4<_Float16>(p);
}
extern "C" __global__ __launch_bounds__(256) void gemv_w4_f32(PhxGemvW4 p) { gemv_w4<float>(p); }
