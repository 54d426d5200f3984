// Copies of pages within pools (phx_pages_copy): a stream of 16-byte loads and
// stores, bound by HBM.  A workgroup moves 16 KiB of one page of one layer,
// four loads of a thread in flight. 200 pages of 68 KiB in 16 layers: 88 us (5.1
// TB/s); 3 pages of 9 KiB: 1.8 us.
#include "phx_common.h"
#include "phx_decode.h"

extern "C" __global__ __launch_bounds__(PHX_PAGES_THREADS) void pages_copy(PhxPagesCopy p) {
    const uint64_t layer = p.pool + blockIdx.z * p.layer_stride;
    const phx_u4 *src = (const phx_u4 *)(layer + p.src[blockIdx.y] * p.page_bytes);
    phx_u4 *dst = (phx_u4 *)(layer + p.dst[blockIdx.y] * p.page_bytes);
    const uint64_t n = p.page_bytes / 16;
    const uint64_t i = (uint64_t)blockIdx.x * (4 * PHX_PAGES_THREADS) + threadIdx.x;
    phx_u4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (i + u * PHX_PAGES_THREADS < n) v[u] = src[i + u * PHX_PAGES_THREADS];
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (i + u * PHX_PAGES_THREADS < n) dst[i + u * PHX_PAGES_THREADS] = v[u];
}
