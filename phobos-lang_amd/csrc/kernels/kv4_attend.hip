// Attention over keys and values held in 4 bits in pages (the layout and the
// arithmetic: include/phobos_hip.h, phx_kv4_attention).
//
// With codes c, scales s and minima m, a key's score and the output are
//   score_j = scale (s_j sum_d q_d c_jd + m_j sum_d q_d)
//   o_d     = (sum_j p_j s_j c_jd + sum_j p_j m_j) / sum_j p_j
// so the codes themselves are the matrix operands, never the values they
// stand for, and the parameters are one multiply-add per key and row.
//
// A wave takes NC tiles of 16 columns, a column being one (row, query head) of
// the KV head, and 32 keys at a time:
//   S (16 keys x 16 columns) = K Q^T      v_mfma_f32_16x16x32_f16, twice
//   O^T (D x 16 columns)    += V^T W^T    W the weights p_j s_j
// The output of the first has a column's keys 4 quad .. 4 quad + 3 in a lane's
// four registers, and the order of the keys inside the second's products is
// free as long as both operands have the same: so a lane's eight weights are
// the second's operand as they stand, and V is stored so that one 16-byte load
// brings the same lane's keys (four tokens' dwords).
//
// A code enters exactly, as an f16 whose mantissa its bits are put into: K's as
// 16 + c (a shift and a mask per pair of codes), the product starting from
// -24 sum_d q_d; V's as 64 + c or 1024 + c less as much and 8 (its sums run over
// all keys: with sizes of 0 .. 15 they would be many times what they leave
// after the minima's term).  Codes as subnormals, 0x000c, would need neither,
// but the matrix instructions keep only about 20 bits of a sum of those
// (measured: errors of 2^-20 of the largest product, 2^-25 with these).
//
// The waves of a workgroup take the key blocks of its share in turns and merge
// at the end in LDS; with too few workgroups for the GPU the keys are split
// further over workgroups, whose results kv4_combine merges.
//
// 64 sequences of 4096 keys, 8 KV heads of 128 with 4 query heads each: 57.7 us,
// the memory's (5.0 TB/s). With less to do it is the vector instructions, 500 for
// 64 keys (unpacking 290, the softmax 110), and a workgroup's start and merge: 32
// sequences of up to 4096 keys, 2100 on average, 25.5 us (2.8 TB/s), the longest
// one's; one sequence of 100003 keys, 4 x 8 heads, 16.6 us and 3.6 to join its 64
// parts.
#include "kv4.h"

#define KV4_LOG2E 1.44269504088896340736f
#define KV4_NONE -3e38f  // a reference below every score: no key yet

namespace {

// Constants kept in registers: with both of its constants as literals, a mask
// and the bits set behind it are two instructions instead of one.
__device__ __forceinline__ uint32_t in_sgpr(uint32_t x) {
    asm("" : "+s"(x));
    return x;
}
__device__ __forceinline__ uint32_t in_vgpr(uint32_t x) {
    asm("" : "+v"(x));
    return x;
}

__device__ __forceinline__ phx_h8 h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(phx_h8, (phx_u4){a, b, c, d});
}
__device__ __forceinline__ phx_f4 mfma(phx_h8 a, phx_h8 b, phx_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ _Float16 half_of(uint32_t w, int i) {
    const phx_h2 h = __builtin_bit_cast(phx_h2, w);
    return i ? h.y : h.x;
}
// What code 8 stands for.
__device__ __forceinline__ float middle(uint32_t w) {
    return fmaf(8.0f, (float)half_of(w, 0), (float)half_of(w, 1));
}
// (scale, minimum) as finite numbers, whatever is in a slot without a token,
// and a scale that is not positive, as of a page never written, as the
// smallest: it stands for the same where codes are 0.
__device__ __forceinline__ uint32_t positive(uint32_t w) {
    const phx_h2 least = {(_Float16)0x1p-24f, (_Float16)-65504.0f};
    const phx_h2 most = {(_Float16)65504.0f, (_Float16)65504.0f};
    return __builtin_bit_cast(
        uint32_t, __builtin_elementwise_min(
                      __builtin_elementwise_max(__builtin_bit_cast(phx_h2, w), least), most));
}

// How a wave's 16 columns are used.  G 1: 16 columns over 32 keys, two products
// of 16 keys.  With at most 16/G columns in the call, G copies of them: copy g
// takes the g-th 16 keys alone.  All copies' scores come out of one chain of
// products, in which the queries of the other copies are zeros, so the softmax
// has 4 scores per lane and none of a column that does not exist, where G 1
// would have 8 per 32 keys.
template <int G>
struct Shape {
    static constexpr int TILES = G == 4 ? 4 : 2;   // of 16 keys, in a step
    static constexpr int UNITS = TILES / 2;        // of 32 keys: what a page holds whole
    static constexpr int SETS = TILES / G;         // of 4 scores per lane
    static constexpr int COLS = 16 / G;
};

// A step's keys as loaded: codes, and (scale, minimum) of the lane's own keys
// 16 t + 4 quad + i, t being its copy's tile (G 1: both).
template <int D, int G>
struct Raw {
    uint32_t k[Shape<G>::TILES][D / 32];
    phx_u4 v[Shape<G>::TILES], kp[Shape<G>::SETS], vp[Shape<G>::SETS];
};

template <typename T>
__device__ __forceinline__ T fetch(const PHX_GLOBAL char *base, uint32_t off) {
    return *(const PHX_GLOBAL T *)(base + off);
}

// Codes of the two tiles of a unit whose head's part of the page is at `head`.
template <int D>
__device__ __forceinline__ void load_k(uint32_t (*to)[D / 32], const PHX_GLOBAL char *head,
                                       uint32_t slot, uint32_t lane) {
    const uint32_t off = (lane & 15) * (D / 2) + (lane >> 4) * (D / 8);
#pragma unroll
    for (int t = 0; t < 2; ++t)
        if constexpr (D == 128) {
            const phx_u4 w = fetch<phx_u4>(head + slot * (D / 2), off + t * 8 * D);
            to[t][0] = w.x, to[t][1] = w.y, to[t][2] = w.z, to[t][3] = w.w;
        } else {
            const phx_u2 w = fetch<phx_u2>(head + slot * (D / 2), off + t * 8 * D);
            to[t][0] = w.x, to[t][1] = w.y;
        }
}
template <int D>
__device__ __forceinline__ void load_v(phx_u4 *to, const PHX_GLOBAL char *head, uint32_t P,
                                       uint32_t slot, uint32_t lane) {
    const uint32_t off = ((lane >> 4) * (D / 8) + (lane & (D / 8 - 1))) * 16;
#pragma unroll
    for (int t = 0; t < 2; ++t) to[t] = fetch<phx_u4>(head + (P + slot) * (D / 2), off + t * 8 * D);
}

// Eight codes of a key as f16: 16 and the code behind it, and for queries of two
// terms 24 less, the middle.  (Sums of 16 + c from -24 sum_d q_d on pass through
// several times their result: f32 outputs of a prompt's chunk were 2.4e-6 off,
// 0.6e-6 without.  For f16 queries, whose outputs round at 2^-11, that saves the
// subtraction.)
template <int TERMS>
__device__ __forceinline__ phx_h8 keys(uint32_t w, uint32_t mask, uint32_t one) {
    const phx_h8 k = h8((w << 6 & mask) | one, (w << 2 & mask) | one, (w >> 2 & mask) | one,
                        (w >> 6 & mask) | one);
    return TERMS == 2 ? k - (_Float16)24 : k;
}

// The columns' queries as matrix operands, and what turns a product into a
// score in log2 units: t = s_j S a + (m_j + 8 s_j) b, S being the product with
// c_j - 8, as it starts at c: with a code's own size 0 .. 15 the
// two terms are larger than their sum and lose its last bits.
template <int D, int TERMS>
struct Query {
    phx_h8 q[TERMS][D / 32];
    float a, b, c;
    int32_t limit;  // keys the column sees
};

template <typename T, int D, int TERMS>
__device__ __forceinline__ void load_query(Query<D, TERMS> &r, const PhxKv4 &p, const Seq &s,
                                           int head, uint32_t col, uint32_t quad) {
    constexpr int N = D / 4;  // elements of a lane: D/4 of a row, from quad D/4 on
    const uint32_t ratio = p.ratio, i = col / ratio;
    const int64_t row = s.row0 + i;
    const bool live = i < s.count && row >= 0 && row < p.rows;
    r.limit = (int32_t)(!live ? 0 : p.causal ? s.tokens - s.count + i + 1 : s.tokens);
    float x[N];
    const PHX_GLOBAL T *src = (const PHX_GLOBAL T *)p.x + row * p.ldx +
                              ((int64_t)head * ratio + col % ratio) * D + quad * N;
#pragma unroll
    for (int u = 0; u < N; u += 16 / sizeof(T)) {
        phx_u4 w = {0, 0, 0, 0};
        if (live) w = *(const PHX_GLOBAL phx_u4 *)(src + u);
#pragma unroll
        for (int i = 0; i < (int)(16 / sizeof(T)); ++i)
            x[u + i] = sizeof(T) == 4 ? __builtin_bit_cast(float, (uint32_t)w[i & 3])
                                      : (float)half_of(w[i / 2 & 3], i & 1);
    }
    float top = 0.0f, sum = 0.0f;
#pragma unroll
    for (int u = 0; u < N; ++u) top = fmaxf(top, fabsf(x[u])), sum += x[u];
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    // the row times a power of two that brings its largest into [2^8, 2^9), so
    // that what f16 cannot hold is below 2^-32 of it
    const int e = top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            // a dword's pairs of nibbles: 0 4, 1 5, 2 6, 3 7
            const float v = ldexpf(x[j * 8 + u / 2 + u % 2 * 4], 9 - e);
            const _Float16 hi = (_Float16)v;
            r.q[0][j][u] = hi;
            if constexpr (TERMS == 2) r.q[1][j][u] = (_Float16)(v - (float)hi);
        }
    r.a = ldexpf(p.scale * KV4_LOG2E, e - 9);
    r.c = TERMS == 2 ? 0.0f : -24.0f * ldexpf(sum, 9 - e);
    // a row with an infinity has no scores, as its weights would be inf / inf
    r.b = top < INFINITY ? sum * (p.scale * KV4_LOG2E) : NAN;
}

// A tile of columns' running state; l and pm of the lane's own keys.
template <int D>
struct State {
    phx_f4 o[D / 16];
    float m, l, pm;
};

// What a lane knows of its copy.
template <int D, int G>
struct Lane {
    uint32_t lane, quad, tile;                     // G 1: tile 0 of each set
    uint32_t keep[G == 1 ? 1 : Shape<G>::TILES];   // all ones for its own tile, else 0
    const phx_h8 *q[G == 1 ? 1 : Shape<G>::TILES]; // queries in LDS, or zeros
};

// x of the lane n columns on, in the same 16.
template <int N>
__device__ __forceinline__ float turned(float x) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x120 + N, 0xf, 0xf, true));
}
// Over a column's copies.
template <int G>
__device__ __forceinline__ float copies_sum(float x) {
    if constexpr (G >= 2) x += turned<8>(x);
    if constexpr (G == 4) x += turned<4>(x);
    return x;
}
template <int G>
__device__ __forceinline__ float copies_max(float x) {
    if constexpr (G >= 2) x = fmaxf(x, turned<8>(x));
    if constexpr (G == 4) x = fmaxf(x, turned<4>(x));
    return x;
}

// The scores' products of a step.
template <int D, int TERMS, int NC, int G>
__device__ __forceinline__ void scores(const Raw<D, G> &r, const Query<D, TERMS> (&q)[NC],
                                       const Lane<D, G> &ln, phx_f4 (&s)[NC][Shape<G>::SETS]) {
    using Sh = Shape<G>;
    const uint32_t mask = in_sgpr(0x03c003c0), one = in_vgpr(0x4c004c00);
    phx_f4 odd = {0, 0, 0, 0};  // G 2, 4: two chains, as one would wait for itself
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int a = 0; a < Sh::SETS; ++a) s[c][a] = (phx_f4){q[c].c, q[c].c, q[c].c, q[c].c};
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int t = 0; t < Sh::TILES; ++t) {
            const uint32_t w = r.k[t][j];
            const phx_h8 k = keys<TERMS>(w, mask, one);
#pragma unroll
            for (int x = 0; x < TERMS; ++x)
                if constexpr (G == 1) {
#pragma unroll
                    for (int c = 0; c < NC; ++c) s[c][t] = mfma(k, q[c].q[x][j], s[c][t]);
                } else {
                    phx_f4 &to = t % 2 ? odd : s[0][0];
                    to = mfma(k, ln.q[t][(x * (D / 32) + j) * 64], to);
                }
        }
    if constexpr (G > 1) s[0][0] = s[0][0] + odd;
}

// The weights p_j s_j of a step's scores, in two f16 terms (22 bits): pairs of
// halves, the f16 of the exact product and of what that leaves.  Keys past what
// a column sees, or in a unit without a page (a bit of `absent`), get zeros.
template <int D, int TERMS, int NC, int G>
__device__ __forceinline__ void weights(const Raw<D, G> &r, const Query<D, TERMS> (&q)[NC],
                                        State<D> (&st)[NC], const Lane<D, G> &ln,
                                        const phx_f4 (&s)[NC][Shape<G>::SETS],
                                        uint32_t (&hi)[NC][2 * Shape<G>::SETS],
                                        uint32_t (&lo)[NC][2 * Shape<G>::SETS], uint32_t key0,
                                        uint32_t absent, bool fresh) {
    constexpr int W = 4 * Shape<G>::SETS;  // scores per lane
    uint32_t vp[W];
    float km[W], vm[W];
#pragma unroll
    for (int u = 0; u < W; ++u) {
        vp[u] = positive(r.vp[u / 4][u % 4]);
        km[u] = middle(r.kp[u / 4][u % 4]);
        vm[u] = middle(vp[u]);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        int32_t left = (int32_t)((uint32_t)q[c].limit - (key0 + 16 * ln.tile + 4 * ln.quad));
        if (absent >> (ln.tile / 2) & 1) left = 0;
        float e[W];
#pragma unroll
        for (int u = 0; u < W; ++u) e[u] = s[c][u / 4][u % 4] * q[c].a;
        // the score in log2 units, less m
        auto score = [&](int u, float m) {
            const float x = fmaf((float)half_of(r.kp[u / 4][u % 4], 0), e[u], fmaf(km[u], q[c].b, -m));
            return 16 * (u / 4) + u % 4 < left ? x : -INFINITY;
        };
        // The reference m is of score + log2 s_V, and stays while no weight
        // passes 40000: rarely raised after the first step, and then to 2^7
        // below the step's largest.  (p itself is at most w 2^24 in f32.  A row
        // with a NaN is NaN whatever its reference.)
        float sum, pm, need = fresh ? INFINITY : 0.0f;
        bool raise = fresh;
        for (int pass = 0; pass < 2; ++pass) {
            if (raise) {
                float most = -INFINITY;
#pragma unroll
                for (int u = 0; u < W; ++u)
                    most = fmaxf(most, score(u, 0.0f) +
                                           __builtin_amdgcn_logf((float)half_of(vp[u], 0)));
                most = copies_max<G>(most);
                most = fmaxf(most, __shfl_xor(most, 16));
                most = fmaxf(most, __shfl_xor(most, 32));
                need = copies_max<G>(need);
                need = fmaxf(need, __shfl_xor(need, 16));
                need = fmaxf(need, __shfl_xor(need, 32));
                // by the column's own weights alone: no row's result depends
                // on the rows next to it
                if (need > 40000.0f && most - 7.0f > st[c].m) {
                    const float f = __builtin_amdgcn_exp2f(st[c].m - (most - 7.0f));
                    st[c].m = most - 7.0f;
                    st[c].l *= f;
                    st[c].pm *= f;
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) st[c].o[j] = st[c].o[j] * f;
                }
            }
            sum = pm = 0.0f;
            phx_h2 h, l, top = {(_Float16)0.0f, (_Float16)0.0f};
#pragma unroll
            for (int u = 0; u < W; ++u) {
                const float pr = __builtin_amdgcn_exp2f(score(u, st[c].m));
                const _Float16 sv = half_of(vp[u], 0);
                sum += pr;
                pm = fmaf(pr, vm[u], pm);
                h[u % 2] = (_Float16)fmaf(pr, (float)sv, 0.0f);
                l[u % 2] = (_Float16)fmaf(pr, (float)sv, -(float)h[u % 2]);
                if (u % 2) {
                    top = __builtin_elementwise_max(top, h);
                    hi[c][u / 2] = __builtin_bit_cast(uint32_t, h);
                    lo[c][u / 2] = __builtin_bit_cast(uint32_t, l);
                }
            }
            need = fmaxf((float)top.x, (float)top.y);
            raise = __any(need > 40000.0f);
            if (!raise) break;
        }
        st[c].l += sum;
        st[c].pm += pm;
    }
}

// The weights' product with a step's values.
template <int D, int NC, int G>
__device__ __forceinline__ void sums(const Raw<D, G> &r, State<D> (&st)[NC], const Lane<D, G> &ln,
                                     const uint32_t (&hi)[NC][2 * Shape<G>::SETS],
                                     const uint32_t (&lo)[NC][2 * Shape<G>::SETS]) {
    const uint32_t mask[2] = {in_sgpr(0x000f000f), in_sgpr(0x00f000f0)};
    const uint32_t one[2] = {in_vgpr(0x64006400), in_vgpr(0x54005400)};
    // an octet of elements per row of the operand; at D 64 the upper eight rows
    // are the same octets' other half
    const uint32_t first = D == 64 && (ln.lane & 8) ? 0x0c060c02 : 0x0c040c00;
#pragma unroll
    for (int n = 0; n < Shape<G>::UNITS; ++n) {
        // the unit's weights: a copy's are zeros but for its own tile
        phx_h8 wh[NC], wl[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if constexpr (G == 1) {
                wh[c] = h8(hi[c][0], hi[c][1], hi[c][2], hi[c][3]);
                wl[c] = h8(lo[c][0], lo[c][1], lo[c][2], lo[c][3]);
            } else {
                const uint32_t k0 = ln.keep[2 * n], k1 = ln.keep[2 * n + 1];
                wh[c] = h8(hi[c][0] & k0, hi[c][1] & k0, hi[c][0] & k1, hi[c][1] & k1);
                wl[c] = h8(lo[c][0] & k0, lo[c][1] & k0, lo[c][0] & k1, lo[c][1] & k1);
            }
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
            const uint32_t sel = first + b * 0x00010001;
            uint32_t x[4];  // a byte of the lane's eight keys, in halves
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const phx_u4 v = r.v[2 * n + t];
                x[2 * t] = __builtin_amdgcn_perm(v.y, v.x, sel);
                x[2 * t + 1] = __builtin_amdgcn_perm(v.w, v.z, sel);
            }
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
                const phx_h8 v = h8((x[0] & mask[odd]) | one[odd], (x[1] & mask[odd]) | one[odd],
                                    (x[2] & mask[odd]) | one[odd], (x[3] & mask[odd]) | one[odd]) -
                                 (_Float16)(odd ? 72 : 1032);
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    st[c].o[2 * b + odd] = mfma(v, wh[c], st[c].o[2 * b + odd]);
                    st[c].o[2 * b + odd] = mfma(v, wl[c], st[c].o[2 * b + odd]);
                }
            }
        }
    }
}

// Four outputs from their sums, zeros without a key.
template <typename T>
__device__ __forceinline__ void store(PHX_GLOBAL T *dst, phx_f4 o, float sum) {
    typedef T four __attribute__((ext_vector_type(4)));
    four out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = (T)(sum == 0.0f ? 0.0f : o[i] / sum);
    *(PHX_GLOBAL four *)dst = out;
}

template <typename T, int D, int NC, int G, int WAVES>
__device__ __forceinline__ void attend(const PhxKv4 &p) {
    using Sh = Shape<G>;
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1, PITCH = D + 4, COLS = NC * Sh::COLS;
    __shared__ float merged[WAVES * Sh::COLS * PITCH];
    __shared__ float stats[WAVES * Sh::COLS * 2];
    __shared__ phx_h8 queries[G == 1 ? 1 : TERMS * (D / 32) * 64 * 2];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Lane<D, G> ln;
    ln.lane = lane;
    ln.quad = lane >> 4;
    ln.tile = G == 1 ? 0 : (lane & 15) / Sh::COLS;
    uint32_t cg = 0, split = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
    if (p.groups > 1) {
        // column groups of one KV head next to each other on one XCD, the
        // longest rows first
        const uint32_t groups = p.groups, splits = p.splits;
        uint32_t item = phx_xcd_swizzle_any(phx_block_linear(), phx_block_count());
        cg = groups - 1 - item % groups;
        item /= groups;
        split = item % splits;
        item /= splits;
        head = item % p.heads;
        b = item / p.heads;
    }
    constexpr uint32_t KEYS = 16 * Sh::TILES, PER = 64 / Sh::UNITS;  // steps of whose pages the lanes hold
    const uint32_t P = p.page_tokens, shift = __builtin_ctz(P / 32);
    const PHX_GLOBAL int32_t *table =
        (const PHX_GLOBAL int32_t *)p.table + b * p.table_stride;
    // the wave's steps are base + WAVES i, and the lanes hold the pages of PER
    // of them; unsplit the first ones are known, and loaded, before the length is
    uint32_t base = __builtin_amdgcn_readfirstlane(wave);
    auto unit_of = [&]() { return (base + lane / Sh::UNITS * WAVES) * Sh::UNITS + lane % Sh::UNITS; };
    int32_t early = -1;
    if (p.splits == 1 && (unit_of() >> shift) < p.table_stride) early = table[unit_of() >> shift];
    const Seq s = kv4_seq(p, b);
    const uint32_t ratio = p.ratio, col0 = cg * COLS, first = col0 / ratio;
    if (first >= s.count) return;
    int64_t last = (col0 + COLS - 1) / ratio;
    if (last >= s.count) last = s.count - 1;
    int64_t most = p.causal ? s.tokens - s.count + last + 1 : s.tokens;  // keys that some column sees
    if (most < 0) most = 0;

    const uint32_t steps = (uint32_t)(most + KEYS - 1) / KEYS;
    const uint32_t per = (steps + p.splits - 1) / p.splits;
    const uint32_t end = min((split + 1) * per, steps);
    const uint32_t units = (uint32_t)(most + 31) / 32;
    base += split * per;
    int32_t ids;
    int n;
    auto pages = [&](bool first) {
        ids = -1;
        const uint32_t mine = unit_of();
        if (base < end && mine < units) ids = first && p.splits == 1 ? early : table[mine >> shift];
        if (ids >= p.pages) ids = -1;
        n = base < end ? min((end - base + WAVES - 1) / WAVES, PER) : 0;
    };
    // a step's page of unit u, and its slot there
    auto slot = [&](int i, int u) {
        return (((base + WAVES * i) * Sh::UNITS + u) & ((1u << shift) - 1)) * 32;
    };
    auto page = [&](int i, int u) {
        const int id = __builtin_amdgcn_readlane(ids, i * Sh::UNITS + u);
        return kv4_head<D>(p, id < 0 ? 0 : id, head);
    };
    Raw<D, G> r;
    auto next_k = [&](int i) {
#pragma unroll
        for (int u = 0; u < Sh::UNITS; ++u) load_k<D>(r.k + 2 * u, page(i, u), slot(i, u), lane);
    };
    auto next_v = [&](int i) {
#pragma unroll
        for (int u = 0; u < Sh::UNITS; ++u)
            load_v<D>(r.v + 2 * u, page(i, u), P, slot(i, u), lane);
    };
    auto next_p = [&](int i) {
        const PHX_GLOBAL char *own = page(i, 0) + slot(i, 0) * 4;
        if (Sh::UNITS == 2 && ln.tile >= 2) own = page(i, 1) + slot(i, 1) * 4;
#pragma unroll
        for (int a = 0; a < Sh::SETS; ++a) {
            const uint32_t off = P * D + (ln.tile % 2 + a) * 64 + ln.quad * 16;
            r.kp[a] = fetch<phx_u4>(own, off);
            r.vp[a] = fetch<phx_u4>(own, off + P * 4);
        }
    };
    // a step's loads go out as the one before is done with their registers, the
    // first step's before the queries are looked at
    auto start = [&](bool first) {
        pages(first);
        if (n == 0) return;
        next_k(0);
        next_p(0);
        next_v(0);
    };
    start(true);

    Query<D, TERMS> q[NC];
    State<D> st[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        load_query<T, D, TERMS>(q[c], p, s, head, col0 + c * 16 + (lane & 15) % Sh::COLS, ln.quad);
        st[c].m = KV4_NONE;
        st[c].l = st[c].pm = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) st[c].o[j] = (phx_f4){0, 0, 0, 0};
    }
    if constexpr (G > 1) {
        // the queries, and as many zeros behind them
        constexpr int N = TERMS * (D / 32);
        if (wave == 0) {
#pragma unroll
            for (int x = 0; x < N; ++x) {
                queries[x * 64 + lane] = q[0].q[x / (D / 32)][x % (D / 32)];
                queries[(N + x) * 64 + lane] = h8(0, 0, 0, 0);
            }
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < Sh::TILES; ++t) {
            const bool own = (uint32_t)t == ln.tile;
            ln.keep[t] = own ? ~0u : 0;
            ln.q[t] = queries + (own ? 0 : N * 64) + lane;
        }
    }
    bool fresh = true;
    while (n > 0) {
        for (int i = 0; i < n; ++i) {
            const uint32_t at = base + WAVES * i;
            uint32_t absent = 0;
#pragma unroll
            for (int u = 0; u < Sh::UNITS; ++u)
                absent |= (__builtin_amdgcn_readlane(ids, i * Sh::UNITS + u) < 0 ? 1u : 0u) << u;
            phx_f4 x[NC][Sh::SETS];
            uint32_t hi[NC][2 * Sh::SETS], lo[NC][2 * Sh::SETS];
            scores<D, TERMS, NC, G>(r, q, ln, x);
            if (i + 1 < n) next_k(i + 1);
            weights<D, TERMS, NC, G>(r, q, st, ln, x, hi, lo, at * KEYS, absent, fresh);
            fresh = false;
            if (i + 1 < n) next_p(i + 1);
            sums<D, NC, G>(r, st, ln, hi, lo);
            if (i + 1 < n) next_v(i + 1);
        }
        base += PER * WAVES;
        start(false);
    }

    // the results of the waves, one tile of columns after the other; a column's
    // copies have one reference
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float l = copies_sum<G>(st[c].l), pm = copies_sum<G>(st[c].pm);
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        pm += __shfl_xor(pm, 16);
        pm += __shfl_xor(pm, 32);
        if (c) __syncthreads();
        const uint32_t col = lane & 15, entry = wave * Sh::COLS + col;
        float *out = merged + entry * PITCH;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t row = 4 * ln.quad + i;
            const uint32_t d = D == 128 ? 8 * row : 8 * (row & 7) + 4 * (row >> 3);
#pragma unroll
            for (int j = 0; j < D / 16; j += 4) {
                phx_f4 o;
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = copies_sum<G>(st[c].o[j + k][i]) + pm;
                if (G == 1 || col < Sh::COLS) *(phx_f4 *)(out + d + j) = o;
            }
        }
        if (lane < Sh::COLS) {
            stats[entry * 2] = st[c].m;
            stats[entry * 2 + 1] = l;
        }
        __syncthreads();
        for (uint32_t x = threadIdx.x; x < Sh::COLS * (D / 4); x += 64 * WAVES) {
            const uint32_t col = x / (D / 4), d = x % (D / 4) * 4;
            float m = KV4_NONE, sum = 0.0f;
            phx_f4 o = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < WAVES; ++w) m = fmaxf(m, stats[(w * Sh::COLS + col) * 2]);
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const uint32_t at = w * Sh::COLS + col;
                const float f = __builtin_amdgcn_exp2f(stats[at * 2] - m);
                sum = fmaf(f, stats[at * 2 + 1], sum);
                const phx_f4 v = *(const phx_f4 *)(merged + at * PITCH + d);
#pragma unroll
                for (int u = 0; u < 4; ++u) o[u] = fmaf(f, v[u], o[u]);
            }
            const uint32_t at = col0 + c * 16 + col, i = at / ratio;
            const int64_t row = s.row0 + i;
            if (i >= s.count || row < 0 || row >= p.rows) continue;
            const int64_t qh = (int64_t)head * ratio + at % ratio;
            if (p.splits == 1) {
                store<T>((PHX_GLOBAL T *)p.y + row * p.ldy + qh * D + d, o, sum);
            } else {
                const int64_t rows = p.rows * p.heads * ratio;
                const int64_t unit = split * rows + row * p.heads * ratio + qh;
                if (sum != 0.0f) *(PHX_GLOBAL phx_f4 *)((PHX_GLOBAL float *)p.ws + unit * D + d) = o;
                if (d == 0) {
                    PHX_GLOBAL float *ml =
                        (PHX_GLOBAL float *)p.ws + rows * p.splits * D + unit * 2;
                    ml[0] = m;
                    ml[1] = sum;
                }
            }
        }
    }
}

// Many columns, as of a prompt's chunk: the work on a key that every column
// repeats, its codes to f16 and its parameters to f32, is done once for a
// workgroup's 128 columns and shared through LDS. Four waves take 32 columns
// each and all of the keys, KEYS at a time; the next ones are loaded while these
// are multiplied, and LDS has two halves, so that there is one barrier in
// between. Bound by the vector instructions: for 32 keys and 32 columns about 220
// of a wave, 110 of them the softmax, next to 48 matrix instructions (2 x 1000
// rows over 4133 keys, 8 x 4 heads of 128: 211 us, 565 TFLOP/s of the products
// without the weights' second term; vector instructions are busy 69 % of the
// cycles, LDS 40 % and the matrix cores 39 %, at two waves a SIMD).
template <int D>
struct Chunk {
    static constexpr int KEYS = 8192 / D;     // 16 KiB of f16 each for K and V
    static constexpr int UNITS = KEYS / 32;
    // K: chunk c of eight elements of key r of tile t at (t D/8 + c) 256 +
    // 16 (r ^ c): reads and writes of 16 lanes touch every bank once (D 64: writes
    // twice).  V: the operand of 16 rows of elements for 32 keys as a wave
    // reads it.
    phx_h8 k[KEYS * D / 8], v[KEYS * D / 8];
    float par[4][KEYS];  // scale and middle of K, of V
};

template <typename T, int D>
__device__ __forceinline__ void chunk(const PhxKv4 &p) {
    using Ch = Chunk<D>;
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1, NC = 2, COLS = 64 * NC;
    constexpr int UNROLL = sizeof(T) == 4 ? 1 : 2;  // as many as fit the registers
    constexpr uint32_t KEYS = Ch::KEYS, UNITS = Ch::UNITS, PER = 64 / UNITS;
    __shared__ Ch lds[2];
    const uint32_t lane = threadIdx.x & 63, quad = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // column groups of one KV head next to each other on one XCD, in turns the
    // longest rows first and last, so that two on a CU differ
    const uint32_t groups = p.groups;
    uint32_t item = phx_xcd_swizzle_any(phx_block_linear(), phx_block_count());
    uint32_t cg = item % groups;
    item /= groups;
    if (item % 2 == 0) cg = groups - 1 - cg;
    const uint32_t head = item % p.heads, b = item / p.heads;
    const Seq s = kv4_seq(p, b);
    const uint32_t ratio = p.ratio, col0 = cg * COLS + wave * (16 * NC);
    if (cg * COLS / ratio >= s.count) return;
    int64_t last = (cg * COLS + COLS - 1) / ratio;
    if (last >= s.count) last = s.count - 1;
    // keys that some column sees, and that all of the wave's columns see
    int64_t most = p.causal ? s.tokens - s.count + last + 1 : s.tokens;
    int64_t least = p.causal ? s.tokens - s.count + col0 / ratio + 1 : s.tokens;
    if (most < 0) most = 0;
    if (least < 0) least = 0;
    const uint32_t steps = (uint32_t)(most + KEYS - 1) / KEYS;
    const uint32_t seen = (uint32_t)least / KEYS;
    const uint32_t units = (uint32_t)(most + 31) / 32;
    const uint32_t P = p.page_tokens, shift = __builtin_ctz(P / 32);
    const PHX_GLOBAL int32_t *table =
        (const PHX_GLOBAL int32_t *)p.table + b * p.table_stride;
    // the lanes hold the pages of PER steps from `base` on
    int32_t ids;
    uint32_t base;
    auto pages = [&](uint32_t from) {
        base = from;
        ids = -1;
        const uint32_t mine = base * UNITS + lane;
        if (mine < units) ids = table[mine >> shift];
        if (ids >= p.pages) ids = -1;
    };
    // the wave's share of a step, all of one unit: 16 bytes of K and of V a
    // lane, and the parameters of 64 / UNITS ... keys
    const uint32_t unit = wave * UNITS / 4;
    const uint32_t own = threadIdx.x % (256 / UNITS);  // in the unit
    constexpr uint32_t PARAMS = KEYS / 4;              // keys of a wave's parameters
    phx_u4 raw_k, raw_v;
    uint32_t raw_p;
    auto fetch_step = [&](uint32_t i) {
        const int id = __builtin_amdgcn_readlane(ids, (i - base) * UNITS + unit);
        const uint32_t slot = ((i * UNITS + unit) & ((1u << shift) - 1)) * 32;
        const PHX_GLOBAL char *part = kv4_head<D>(p, id < 0 ? 0 : id, head);
        raw_k = fetch<phx_u4>(part + slot * (D / 2), own * 16);
        raw_v = fetch<phx_u4>(part + (P + slot) * (D / 2), own * 16);
        if (lane < 2 * PARAMS)
            raw_p = fetch<uint32_t>(part, P * D + (lane < PARAMS ? 0 : 4 * P) +
                                              4 * (slot + wave * PARAMS % 32 + lane % PARAMS));
    };
    auto stage = [&](Ch &to) {
        const uint32_t mask = in_sgpr(0x03c003c0), one = in_vgpr(0x4c004c00);
        constexpr uint32_t LANES = D / 32;  // of a key
        const uint32_t key = threadIdx.x / LANES, r = key & 15;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t w = raw_k[i], c = threadIdx.x % LANES * 4 + i;
            to.k[(key / 16 * (D / 8) + c) * 16 + ((r ^ c) & 15)] =
                keys<TERMS>(w, mask, one);
        }
        // four keys' dwords of octet e: halves of the operands' 16 bytes
        const uint32_t low[2] = {in_sgpr(0x000f000f), in_sgpr(0x00f000f0)};
        const uint32_t bits[2] = {in_vgpr(0x64006400), in_vgpr(0x54005400)};
        const uint32_t four = threadIdx.x / (D / 8), e = threadIdx.x % (D / 8);
        phx_u2 *dst = (phx_u2 *)to.v + ((four / 8 * (D / 16)) * 64 + four % 4 * 16 + e) * 2 + four / 4 % 2;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            const uint32_t sel = 0x0c040c00 + x / 2 * 0x00010001;
            const uint32_t a = __builtin_amdgcn_perm(raw_v.y, raw_v.x, sel);
            const uint32_t c = __builtin_amdgcn_perm(raw_v.w, raw_v.z, sel);
            typedef _Float16 h4 __attribute__((ext_vector_type(4)));
            const h4 v = __builtin_bit_cast(h4, (phx_u2){(a & low[x % 2]) | bits[x % 2],
                                                         (c & low[x % 2]) | bits[x % 2]}) -
                         (_Float16)(x % 2 ? 72 : 1032);
            dst[D == 128 ? x * 128 : (x % 4 * 64 + x / 4 * 8) * 2] = __builtin_bit_cast(phx_u2, v);
        }
        if (lane < 2 * PARAMS) {
            const bool values = lane >= PARAMS;
            const uint32_t w = values ? positive(raw_p) : raw_p;
            const uint32_t key = wave * PARAMS + lane % PARAMS;
            to.par[values ? 2 : 0][key] = (float)half_of(w, 0);
            to.par[values ? 3 : 1][key] = middle(w);
        }
    };
    pages(0);
    if (steps > 0) fetch_step(0);

    Query<D, TERMS> q[NC];
    State<D> st[NC];
    phx_f4 zero[NC];
    bool none[NC];  // the column sees keys, but none so far
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        load_query<T, D, TERMS>(q[c], p, s, head, col0 + c * 16 + (lane & 15), quad);
        zero[c] = (phx_f4){q[c].c, q[c].c, q[c].c, q[c].c};
        none[c] = q[c].limit > 0;
        st[c].m = st[c].l = st[c].pm = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) st[c].o[j] = (phx_f4){0, 0, 0, 0};
    }
    for (uint32_t at = 0; at < steps; ++at) {
        Ch &now = lds[at % 2];
        uint32_t absent = 0;  // units without a page
#pragma unroll
        for (uint32_t u = 0; u < UNITS; ++u)
            absent |= (__builtin_amdgcn_readlane(ids, (at - base) * UNITS + u) < 0 ? 1u : 0u) << u;
        stage(now);
        __syncthreads();
        if (at + 1 < steps) {
            if (at + 1 - base == PER) pages(at + 1);
            fetch_step(at + 1);
        }
#pragma unroll UNROLL
        for (uint32_t n = 0; n < UNITS; ++n) {
            // a lane's scores: columns 16 c + lane % 16, keys 16 t + 4 quad + i
            phx_f4 x[NC][2], ks[2], km[2], vs[2], vm[2];
#pragma unroll
            for (int j = 0; j < D / 32; ++j)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint32_t o = quad * (D / 32) + j;
                    const phx_h8 k = now.k[((2 * n + t) * (D / 8) + o) * 16 + ((lane ^ o) & 15)];
#pragma unroll
                    for (int y = 0; y < TERMS; ++y)
#pragma unroll
                        for (int c = 0; c < NC; ++c)
                            x[c][t] = mfma(k, q[c].q[y][j], j || y ? x[c][t] : zero[c]);
                }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint32_t key = n * 32 + t * 16 + quad * 4;
                ks[t] = *(const phx_f4 *)&now.par[0][key];
                km[t] = *(const phx_f4 *)&now.par[1][key];
                vs[t] = *(const phx_f4 *)&now.par[2][key];
                vm[t] = *(const phx_f4 *)&now.par[3][key];
            }
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    x[c][u / 4][u % 4] = fmaf(ks[u / 4][u % 4], x[c][u / 4][u % 4] * q[c].a,
                                              fmaf(km[u / 4][u % 4], q[c].b, -st[c].m));
            if (at >= seen || absent) {
                const uint32_t key0 = at * KEYS + n * 32 + quad * 4;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int32_t left =
                        absent >> n & 1 ? 0 : (int32_t)((uint32_t)q[c].limit - key0);
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        x[c][u / 4][u % 4] =
                            16 * (u / 4) + u % 4 < left ? x[c][u / 4][u % 4] : -INFINITY;
                }
            }
            // as weights() has it, with the scores kept less m
            __builtin_amdgcn_s_setprio(1);  // before the products of the wave next to it
            uint32_t hi[NC][4], lo[NC][4];
            float sum[NC], pm[NC], need[NC];
            auto weigh = [&]() {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    phx_h2 h, l, top = {(_Float16)0.0f, (_Float16)0.0f};
                    sum[c] = pm[c] = 0.0f;
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const float pr = __builtin_amdgcn_exp2f(x[c][u / 4][u % 4]);
                        const float sv = vs[u / 4][u % 4];
                        sum[c] += pr;
                        pm[c] = fmaf(pr, vm[u / 4][u % 4], pm[c]);
                        h[u % 2] = (_Float16)fmaf(pr, sv, 0.0f);
                        l[u % 2] = (_Float16)fmaf(pr, sv, -(float)h[u % 2]);
                        if (u % 2) {
                            top = __builtin_elementwise_max(top, h);
                            hi[c][u / 2] = __builtin_bit_cast(uint32_t, h);
                            lo[c][u / 2] = __builtin_bit_cast(uint32_t, l);
                        }
                    }
                    need[c] = none[c] ? INFINITY : fmaxf((float)top.x, (float)top.y);
                }
            };
            weigh();
            bool raise = false;
#pragma unroll
            for (int c = 0; c < NC; ++c) raise |= need[c] > 40000.0f;
            if (__any(raise)) {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    float most = -INFINITY;
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        most = fmaxf(most,
                                     x[c][u / 4][u % 4] + __builtin_amdgcn_logf(vs[u / 4][u % 4]));
                    most = fmaxf(most, __shfl_xor(most, 16));
                    most = fmaxf(most, __shfl_xor(most, 32));
                    need[c] = fmaxf(need[c], __shfl_xor(need[c], 16));
                    need[c] = fmaxf(need[c], __shfl_xor(need[c], 32));
                    if (need[c] > 40000.0f && most > (none[c] ? -INFINITY : 7.0f)) {
                        const float up = most - 7.0f;
                        const float f = none[c] ? 0.0f : __builtin_amdgcn_exp2f(-up);
                        none[c] = false;
                        st[c].m += up;
                        st[c].l *= f;
                        st[c].pm *= f;
#pragma unroll
                        for (int j = 0; j < D / 16; ++j) st[c].o[j] = st[c].o[j] * f;
#pragma unroll
                        for (int t = 0; t < 2; ++t) x[c][t] = x[c][t] - up;
                    }
                }
                weigh();
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                st[c].l += sum[c];
                st[c].pm += pm[c];
            }
            __builtin_amdgcn_s_setprio(0);
            const phx_h8 *v = now.v + n * (D / 16) * 64 + lane;
#pragma unroll
            for (int j = 0; j < D / 16; j += 2) {
                // a sum's two products apart, as the second waits for the first
                const phx_h8 w[2] = {v[j * 64], v[(j + 1) * 64]};
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int c = 0; c < NC; ++c) {
                            const uint32_t(&r)[4] = y ? lo[c] : hi[c];
                            st[c].o[j + k] = mfma(w[k], h8(r[0], r[1], r[2], r[3]), st[c].o[j + k]);
                        }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float l = st[c].l, pm = st[c].pm;
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        pm += __shfl_xor(pm, 16);
        pm += __shfl_xor(pm, 32);
        const uint32_t col = col0 + c * 16 + (lane & 15), i = col / ratio;
        const int64_t row = s.row0 + i;
        if (i >= s.count || row < 0 || row >= p.rows) continue;
        const int64_t qh = (int64_t)head * ratio + col % ratio;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t r = 4 * quad + i;
            const uint32_t d = D == 128 ? 8 * r : 8 * (r & 7) + 4 * (r >> 3);
#pragma unroll
            for (int j = 0; j < D / 16; j += 4) {
                phx_f4 o;
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = st[c].o[j + k][i] + pm;
                store<T>((PHX_GLOBAL T *)p.y + row * p.ldy + qh * D + d + j, o, l);
            }
        }
    }
}

// The parts of a split launch: a workgroup per row and query head, D/4 lanes by
// 2048/D, each of which takes up to PARTS parts, in a fixed order. All parts are
// loaded before the statistics that weigh them have come: latency is all that
// this costs (32 rows of 64 parts 3.6 us; with the statistics first and four
// parts at a time 5.4).
template <typename T, int D>
__device__ __forceinline__ void combine(const PhxKv4 &p) {
    constexpr int L = D / 4, G = 512 / L, PARTS = PHX_KV4_SPLITS / G;
    __shared__ float factor[PHX_KV4_SPLITS];
    __shared__ float part_m[2], part_l[2];
    __shared__ phx_f4 sums[G][L];
    const uint32_t heads = p.heads * p.ratio, max_q = (uint32_t)p.max_q;
    const uint32_t qh = blockIdx.x % heads, i = blockIdx.x / heads % max_q;
    const Seq s = kv4_seq(p, blockIdx.x / heads / max_q);
    const int64_t row = s.row0 + i;
    if (i >= s.count || row < 0 || row >= p.rows) return;
    const int64_t units = p.rows * heads, unit = row * heads + qh;
    const int t = threadIdx.x, g = t / L, lane = t % L;
    const PHX_GLOBAL float *part = (const PHX_GLOBAL float *)p.ws + unit * D + lane * 4;
    phx_f4 v[PARTS];
#pragma unroll
    for (int x = 0; x < PARTS; ++x)
        if (g + x * G < p.splits) v[x] = *(const PHX_GLOBAL phx_f4 *)(part + (g + x * G) * units * D);
    float m = KV4_NONE, l = 0.0f;
    if (t < p.splits) {
        const PHX_GLOBAL float *w =
            (const PHX_GLOBAL float *)p.ws + units * p.splits * D + (t * units + unit) * 2;
        l = w[1];
        if (l != 0.0f) m = w[0];
    }
    float top = m;
    for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    if (t < PHX_KV4_SPLITS && (t & 63) == 0) part_m[t >> 6] = top;
    __syncthreads();
    top = fmaxf(part_m[0], part_m[1]);
    // a part without keys has stored no sums: its factor of 0 leaves them out
    const float f = l != 0.0f ? __builtin_amdgcn_exp2f(m - top) : 0.0f;
    if (t < PHX_KV4_SPLITS) factor[t] = f;
    float sum = f * l;
    for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
    if (t < PHX_KV4_SPLITS && (t & 63) == 0) part_l[t >> 6] = sum;
    __syncthreads();
    phx_f4 o = {0, 0, 0, 0};
#pragma unroll
    for (int x = 0; x < PARTS; ++x) {
        if (g + x * G >= p.splits) continue;
        const float w = factor[g + x * G];
        if (w == 0.0f) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(w, v[x][e], o[e]);
    }
    sums[g][lane] = o;
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int x = 1; x < G; ++x) o = o + sums[x][lane];
    store<T>((PHX_GLOBAL T *)p.y + row * p.ldy + qh * D + lane * 4, o, part_l[0] + part_l[1]);
}

}  // namespace

#define ATTEND(T, D, suffix, NC, G, WAVES, PER_SIMD)                                            \
    extern "C" __global__ __launch_bounds__(64 * WAVES, PER_SIMD) void                          \
        kv4_attend_##suffix##_c##NC##_g##G##_w##WAVES(PhxKv4 p) {                               \
        attend<T, D, NC, G, WAVES>(p);                                                          \
    }
#define CHUNK(T, D, suffix)                                                                     \
    extern "C" __global__ __launch_bounds__(256, 2) void kv4_attend_##suffix##_chunk(PhxKv4 p) {\
        chunk<T, D>(p);                                                                         \
    }
#define COMBINE(T, D, suffix)                                                                   \
    extern "C" __global__ __launch_bounds__(512) void kv4_combine_##suffix(PhxKv4 p) {          \
        combine<T, D>(p);                                                                       \
    }
// (f32, D 64, c1_g2_w16 spills 7 of its 128 registers, no other one any.)
#define ALL(T, D, suffix)                                                                       \
    ATTEND(T, D, suffix, 1, 4, 4, 2)                                                            \
    ATTEND(T, D, suffix, 1, 2, 4, 2)                                                            \
    ATTEND(T, D, suffix, 1, 1, 4, 2)                                                            \
    ATTEND(T, D, suffix, 1, 4, 12, 3)                                                           \
    ATTEND(T, D, suffix, 1, 2, 16, 4)                                                           \
    ATTEND(T, D, suffix, 1, 1, 8, 2)                                                            \
    CHUNK(T, D, suffix)                                                                         \
    COMBINE(T, D, suffix)
ALL(_Float16, 64, f16_d64)
ALL(_Float16, 128, f16_d128)
ALL(float, 64, f32_d64)
ALL(float, 128, f32_d128)
ATTEND(_Float16, 64, f16_d64, 2, 1, 4, 2)
ATTEND(_Float16, 128, f16_d128, 2, 1, 4, 2)
ATTEND(float, 64, f32_d64, 2, 1, 4, 2)
ATTEND(float, 128, f32_d128, 2, 1, 4, 1)
