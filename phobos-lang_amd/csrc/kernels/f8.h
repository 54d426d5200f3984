// e4m3 codes of f32 values: of t in a block of largest magnitude a, the code of
// 448 t / a (include/phobos_hip.h, "rows and weights in 8 bits").
#pragma once
#include "phx_common.h"
#include "phx_f8.h"

// Addresses arrive as integers: without their address space they would be
// accessed with flat instructions, which also take the LDS path.
#define PHX_GLOBAL __attribute__((address_space(1)))

namespace {

// The magnitude's bits: as whole numbers they order magnitudes, infinity above
// the finite ones and NaN above infinity, so that a maximum keeps both.
__device__ __forceinline__ uint32_t f8_magnitude(float t) {
    return __builtin_bit_cast(uint32_t, t) & 0x7fffffffu;
}

// q rounded to f32 such that rounding it on to a shorter format rounds q itself:
// cut towards zero, with the last bit set where something was cut off.
__device__ __forceinline__ float f8_odd(double q) {
    uint32_t bits = __builtin_bit_cast(uint32_t, (float)q);
    const double back = (double)__builtin_bit_cast(float, bits);
    if (back != q) {
        if (fabs(back) > fabs(q)) bits -= 1;
        bits |= 1;
    }
    return __builtin_bit_cast(float, bits);
}

// Codes of N values (a multiple of 4), four a dword, and `a` the magnitude of
// their block's largest.
template <int N>
__device__ __forceinline__ void f8_codes(const float (&t)[N], uint32_t a, uint32_t (&out)[N / 4]) {
    const float big = __builtin_bit_cast(float, a);
    // 448 / a to 2^-22 of it; NaN where a is no number or infinite, 0 where it is 0
    float inverse = 448.0f * __builtin_amdgcn_rcpf(big);
    if (a >= 0x7f800000u) inverse = __builtin_nanf("");
    if (a == 0) inverse = 0.0f;
    // Outside of 2^-100 .. 2^100 the reciprocal or the quotient leaves f32's range.
    bool again = a != 0 && a < 0x7f800000u && a - 0x0d800000u > 0x64000000u;
    float q[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        q[i] = t[i] * inverse;
        // The quotient is 2^-21.4 of itself off at most: nearer than 16 of its last
        // bits to the middle of two codes it is taken again in 64 bits.  Codes below
        // 2^-6 are 2^-9 apart, as those of 2^-6 and up.
        const float m = fabsf(q[i]), v = m < 0x1p-6f ? m + 0x1p-6f : m;
        again |= ((__builtin_bit_cast(uint32_t, v) & 0xfffffu) - 0x7fff0u) <= 0x20u;
    }
    if (again && a < 0x7f800000u && a != 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = f8_odd(448.0 * (double)t[i] / (double)big);
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
        out[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], w, true);
    }
}

}  // namespace
