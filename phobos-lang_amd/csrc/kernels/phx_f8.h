// What the host runtime and the kernels over 8-bit rows and weights (f8_rows.hip,
// gemm_f8.hip) share: their argument records and launch geometry.
#pragma once
#include <stdint.h>

#define PHX_F8_BLOCK 128  // elements of a row, or rows and elements of a weight, to a scale
#define PHX_F8_NORM_MOST 32768  // elements of a row of the norm

// The kernels that write 8-bit rows.  Element strides; of x, r, h and y those that
// are 0 are not there.
struct PhxF8Rows {
    uint64_t x, r, gain, h, y, q, scales;
    int64_t M, K, ldx, ldr, ldh, ldy, ldq, lds;
    double inverse;  // 1 / K
    float eps;
};

// The products: C's M rows, of A's `rows`.
struct PhxF8Gemm {
    uint64_t a, sa, w, sw, c, starts, list;
    int64_t M, N, K, rows, lda, lds, ldc, experts;
    float alpha, beta;
};
