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
// A code enters as the f16 with its bits: 0x000c is c 2^-24, 0x00c0 is c 2^-20,
// both exact (the matrix instructions keep f16 subnormals).  So unpacking is a
// mask (and for half of them a shift or a byte permute) per pair of codes, and
// no subtraction; the powers of two go into the queries and the last scaling.
//
// The waves of a workgroup take the key blocks of its share in turns and merge
// at the end in LDS; with too few workgroups for the GPU the keys are split
// further over workgroups, whose results kv4_combine merges.
#include "kv4.h"

#define KV4_WAVES 4
#define KV4_LOG2E 1.44269504088896340736f
#define KV4_NONE -3e38f  // a reference below every score: no key yet

namespace {

constexpr uint32_t kLow = 0x000f000f, kHigh = 0x00f000f0, kBias = 0x64006400;

__device__ __forceinline__ phx_h8 h8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(phx_h8, (phx_u4){a, b, c, d});
}
// Halves of 1024 + x, less `off`: exact, as every whole number up to 2048 is.
__device__ __forceinline__ phx_h8 centred(uint32_t a, uint32_t b, uint32_t c, uint32_t d,
                                          int off) {
    const phx_h8 v = h8(a | kBias, b | kBias, c | kBias, d | kBias);
    return v - (_Float16)off;
}
__device__ __forceinline__ phx_f4 mfma(phx_h8 a, phx_h8 b, phx_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ _Float16 half_of(uint32_t w, int i) {
    const phx_h2 h = __builtin_bit_cast(phx_h2, w);
    return i ? h.y : h.x;
}

// 32 keys as loaded: codes, and (scale, minimum) of the lane's keys
// 16 t + 4 quad + i.
template <int D>
struct Raw {
    uint32_t k[2][D / 32];
    phx_u4 v[2], kp[2], vp[2];
};

template <int D>
__device__ __forceinline__ void load_block(Raw<D> &r, const char *head, uint32_t P, uint32_t slot,
                                           uint32_t lane) {
    const uint32_t c = lane & 15, quad = lane >> 4;
    const char *k = head + slot * (D / 2), *v = k + P * (D / 2);
    const char *kp = head + P * D + slot * 4, *vp = kp + P * 4;
    const uint32_t ko = c * (D / 2) + quad * (D / 8);
    const uint32_t vo = (quad * (D / 8) + (c & (D / 8 - 1))) * 16;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        if constexpr (D == 128) {
            const phx_u4 w = *(const phx_u4 *)(k + ko + t * 8 * D);
            r.k[t][0] = w.x, r.k[t][1] = w.y, r.k[t][2] = w.z, r.k[t][3] = w.w;
        } else {
            const phx_u2 w = *(const phx_u2 *)(k + ko + t * 8 * D);
            r.k[t][0] = w.x, r.k[t][1] = w.y;
        }
        r.v[t] = *(const phx_u4 *)(v + vo + t * 8 * D);
        r.kp[t] = *(const phx_u4 *)(kp + quad * 16 + t * 64);
        r.vp[t] = *(const phx_u4 *)(vp + quad * 16 + t * 64);
    }
}

// The columns' queries as matrix operands, and what turns a product into a
// score in log2 units: t = s_j x S x a + m_j x b.
template <int D, int TERMS>
struct Query {
    phx_h8 q[TERMS][D / 32];
    float a, b;
    int32_t limit;  // keys the column sees
};

template <typename T, int D, int TERMS>
__device__ __forceinline__ void load_query(Query<D, TERMS> &r, const PhxKv4 &p, const Seq &s,
                                           int head, int64_t col, uint32_t quad) {
    constexpr int N = D / 4;  // elements of a lane: D/4 of a row, from quad D/4 on
    const int64_t i = col / p.ratio, row = s.row0 + i;
    const bool live = i < s.count && row >= 0 && row < p.rows;
    r.limit = (int32_t)(!live ? 0 : p.causal ? s.tokens - s.count + i + 1 : s.tokens);
    float x[N];
    const T *src = (const T *)p.x + row * p.ldx +
                   ((int64_t)head * p.ratio + col % p.ratio) * D + quad * N;
#pragma unroll
    for (int u = 0; u < N; u += 16 / sizeof(T)) {
        phx_u4 w = {0, 0, 0, 0};
        if (live) w = *(const phx_u4 *)(src + u);
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
            // element of the pair of dwords: nibbles 0 4 2 6 (the even operand,
            // 16 below the odd one, 1 5 3 7)
            constexpr int order[4] = {0, 4, 2, 6};
            const int d = (j / 2) * 16 + (u / 4) * 8 + order[u % 4] + (j & 1);
            const float v = ldexpf(x[d], 9 - e + (j & 1 ? 0 : 4));
            const _Float16 hi = (_Float16)v;
            r.q[0][j][u] = hi;
            if constexpr (TERMS == 2) r.q[1][j][u] = (_Float16)(v - (float)hi);
        }
    r.a = ldexpf(p.scale * KV4_LOG2E, 11 + e);
    // a row with an infinity has no scores, as its weights would be inf / inf
    r.b = top < INFINITY ? sum * (p.scale * KV4_LOG2E) : NAN;
}

// A tile of columns' running state; l and pm of the lane's own keys.
template <int D>
struct State {
    phx_f4 o[D / 16];
    float m, l, pm;
};

template <int D, int TERMS, int NC, bool MASK>
__device__ __forceinline__ void attend_block(const Raw<D> &r, const Query<D, TERMS> (&q)[NC],
                                             State<D> (&st)[NC], uint32_t key0, uint32_t lane) {
    const uint32_t quad = lane >> 4;
    phx_h8 k[2][D / 32], v[D / 16];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < D / 64; ++u) {
            const uint32_t a = r.k[t][2 * u], b = r.k[t][2 * u + 1];
            k[t][2 * u] = h8(a & kLow, (a >> 8) & kLow, b & kLow, (b >> 8) & kLow);
            k[t][2 * u + 1] = h8(a & kHigh, (a >> 8) & kHigh, b & kHigh, (b >> 8) & kHigh);
        }
    // an octet of elements per row of the operand; at D 64 the upper eight rows
    // are the same octets' other half
    const uint32_t first = D == 64 && (lane & 8) ? 0x0c060c02 : 0x0c040c00;
#pragma unroll
    for (int b = 0; b < D / 32; ++b) {
        const uint32_t sel = first + b * 0x00010001;
        uint32_t x[4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            x[2 * t] = __builtin_amdgcn_perm(r.v[t].y, r.v[t].x, sel);
            x[2 * t + 1] = __builtin_amdgcn_perm(r.v[t].w, r.v[t].z, sel);
        }
        v[2 * b] = centred(x[0] & kLow, x[1] & kLow, x[2] & kLow, x[3] & kLow, 1032);
        v[2 * b + 1] = centred(x[0] & kHigh, x[1] & kHigh, x[2] & kHigh, x[3] & kHigh, 1152);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int32_t left = q[c].limit - (int32_t)(key0 + 4 * quad);
        phx_f4 s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t] = (phx_f4){0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < D / 32; ++j)
#pragma unroll
                for (int x = 0; x < TERMS; ++x) s[t] = mfma(k[t][j], q[c].q[x][j], s[t]);
        }
        float w[8], low[8], sum = 0.0f, pm = 0.0f, top = 0.0f;
        // weights against the reference m; their largest tells whether it holds
        auto weigh = [&]() {
            sum = pm = top = 0.0f;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int t = u / 4, i = u % 4;
                const float x = (float)half_of(r.kp[t][i], 0) * s[t][i];
                const float y = fmaf((float)half_of(r.kp[t][i], 1), q[c].b, -st[c].m);
                float e = fmaf(x, q[c].a, y);
                float sv = fmaxf((float)half_of(r.vp[t][i], 0), 0x1p-24f);
                float mv = fmaf(8.0f, sv, (float)half_of(r.vp[t][i], 1));
                if (MASK) {
                    const bool in = 16 * t + i < left;
                    e = in ? e : -INFINITY;
                    sv = in ? sv : 0.0f;
                    mv = in ? mv : 0.0f;
                }
                const float pr = __builtin_amdgcn_exp2f(e);
                w[u] = pr * sv;
                sum += pr;
                pm = fmaf(pr, mv, pm);
                top = fmaxf(top, w[u] == w[u] ? w[u] : INFINITY);
            }
        };
        weigh();
        // The reference m is of score + log2 s_V, and stays while no weight
        // passes 2^15: rarely raised after the first block, and then to 2^7
        // below the block's largest.  (p itself is at most w 2^24 in f32.)
        if (__any(!(top <= 32768.0f))) {
            float most = -INFINITY;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int t = u / 4, i = u % 4;
                const float x = (float)half_of(r.kp[t][i], 0) * s[t][i];
                const float e = fmaf(x, q[c].a, (float)half_of(r.kp[t][i], 1) * q[c].b);
                const float sv = fmaxf((float)half_of(r.vp[t][i], 0), 0x1p-24f);
                const bool in = !MASK || 16 * t + i < left;
                most = fmaxf(most, in ? e + __builtin_amdgcn_logf(sv) : -INFINITY);
            }
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            // by the column's own weights alone: no row's result depends on
            // the rows next to it
            if (top > 32768.0f && most - 7.0f > st[c].m) {
                const float f = __builtin_amdgcn_exp2f(st[c].m - (most - 7.0f));
                st[c].m = most - 7.0f;
                st[c].l *= f;
                st[c].pm *= f;
#pragma unroll
                for (int j = 0; j < D / 16; ++j) st[c].o[j] = st[c].o[j] * f;
            }
            weigh();
        }
        st[c].l += sum;
        st[c].pm += pm;
        // weights in two f16 terms: 22 bits
        phx_h8 hi, lo;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            hi[u] = (_Float16)w[u];
            lo[u] = (_Float16)(w[u] - (float)hi[u]);
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            st[c].o[j] = mfma(v[j], hi, st[c].o[j]);
            st[c].o[j] = mfma(v[j], lo, st[c].o[j]);
        }
    }
}

// N outputs from their sums, zeros without a key.
template <typename T, int N>
__device__ __forceinline__ void store(T *dst, const float (&o)[N], float sum) {
    T out[N];
#pragma unroll
    for (int u = 0; u < N; ++u) out[u] = (T)(sum == 0.0f ? 0.0f : o[u] / sum);
    __builtin_memcpy(__builtin_assume_aligned(dst, N * sizeof(T) < 16 ? N * sizeof(T) : 16), out,
                     sizeof out);
}

template <typename T, int D, int NC>
__device__ __forceinline__ void attend(const PhxKv4 &p) {
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1, PITCH = D + 4;
    __shared__ float merged[KV4_WAVES * 16 * PITCH];
    __shared__ float stats[KV4_WAVES * 16 * 2];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quad = lane >> 4;
    // column groups of one KV head next to each other, and so on one XCD
    int64_t item = phx_xcd_swizzle_any(blockIdx.x, gridDim.x);
    const int64_t groups = (p.max_q * p.ratio + 16 * NC - 1) / (16 * NC);
    const int64_t cg = groups - 1 - item % groups;  // the longest rows first
    item /= groups;
    const uint32_t split = (uint32_t)(item % p.splits);
    item /= p.splits;
    const int head = (int)(item % p.heads);
    const int64_t b = item / p.heads;
    const Seq s = kv4_seq(p, b);
    const int64_t col0 = cg * 16 * NC, first = col0 / p.ratio;
    if (first >= s.count) return;
    int64_t last = (col0 + 16 * NC - 1) / p.ratio;
    if (last >= s.count) last = s.count - 1;
    // keys that some column sees, and that all columns with a row see
    int64_t most = p.causal ? s.tokens - s.count + last + 1 : s.tokens;
    int64_t least = p.causal ? s.tokens - s.count + first + 1 : s.tokens;
    if (most < 0) most = 0;
    if (least < 0) least = 0;

    Query<D, TERMS> q[NC];
    State<D> st[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        load_query<T, D, TERMS>(q[c], p, s, head, col0 + c * 16 + (lane & 15), quad);
        st[c].m = KV4_NONE;
        st[c].l = st[c].pm = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) st[c].o[j] = (phx_f4){0, 0, 0, 0};
    }
    const uint32_t blocks = (uint32_t)(most + 31) / 32;  // fewer than 2^26
    const uint32_t per = (blocks + p.splits - 1) / p.splits;
    const uint32_t end = min((split + 1) * per, blocks);
    const uint32_t P = p.page_tokens, shift = __builtin_ctz(P / 32);
    const int32_t *table = (const int32_t *)p.table + b * p.table_stride;
    // the wave's blocks are begin + KV4_WAVES i; the lanes hold the pages of 64
    // of them
    const uint32_t begin = split * per + __builtin_amdgcn_readfirstlane(wave);
    for (uint32_t base = begin; base < end; base += 64 * KV4_WAVES) {
        int32_t ids = -1;
        const uint32_t mine = base + KV4_WAVES * lane;
        if (mine < end) ids = table[mine >> shift];
        if (ids >= p.pages) ids = -1;
        const int n = min((end - base + KV4_WAVES - 1) / KV4_WAVES, 64u);
        auto where = [&](int i) {
            const int id = __builtin_amdgcn_readlane(ids, i);
            return kv4_head<D>(p, id < 0 ? 0 : id, head);
        };
        auto slot = [&](int i) { return ((base + KV4_WAVES * i) & ((1u << shift) - 1)) * 32; };
        Raw<D> next;
        load_block<D>(next, where(0), P, slot(0), lane);
        for (int i = 0; i < n; ++i) {
            const Raw<D> now = next;
            if (i + 1 < n) load_block<D>(next, where(i + 1), P, slot(i + 1), lane);
            if (__builtin_amdgcn_readlane(ids, i) < 0) continue;
            const uint32_t key0 = (base + KV4_WAVES * i) * 32;
            if (key0 + 32 <= (uint32_t)least)
                attend_block<D, TERMS, NC, false>(now, q, st, key0, lane);
            else
                attend_block<D, TERMS, NC, true>(now, q, st, key0, lane);
        }
    }

    // the waves' results of one tile of columns after the other
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float l = st[c].l, pm = st[c].pm;
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        pm += __shfl_xor(pm, 16);
        pm += __shfl_xor(pm, 32);
        if (c) __syncthreads();
        float *out = merged + (wave * 16 + (lane & 15)) * PITCH;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t row = 4 * quad + i;
            const uint32_t d = D == 128 ? 8 * row : 8 * (row & 7) + 4 * (row >> 3);
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
                out[d + j] = fmaf(st[c].o[j][i], j & 1 ? 0x1p-4f : 1.0f, pm);
        }
        if (quad == 0) {
            stats[(wave * 16 + lane) * 2] = st[c].m;
            stats[(wave * 16 + lane) * 2 + 1] = l;
        }
        __syncthreads();
        // 16 threads per column, D/16 elements each
        constexpr int N = D / 16;
        const uint32_t col = threadIdx.x >> 4, d = (threadIdx.x & 15) * N;
        float m = stats[col * 2], sum = 0.0f, o[N] = {};
#pragma unroll
        for (int w = 1; w < KV4_WAVES; ++w) m = fmaxf(m, stats[(w * 16 + col) * 2]);
#pragma unroll
        for (int w = 0; w < KV4_WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(stats[(w * 16 + col) * 2] - m);
            sum = fmaf(f, stats[(w * 16 + col) * 2 + 1], sum);
#pragma unroll
            for (int u = 0; u < N; ++u)
                o[u] = fmaf(f, merged[(w * 16 + col) * PITCH + d + u], o[u]);
        }
        const int64_t at = col0 + c * 16 + col, i = at / p.ratio, row = s.row0 + i;
        if (i >= s.count || row < 0 || row >= p.rows) continue;
        const int64_t qh = (int64_t)head * p.ratio + at % p.ratio;
        if (p.splits == 1) {
            T *dst = (T *)p.y + row * p.ldy + qh * D + d;
            store<T, N>(dst, o, sum);
        } else {
            const int64_t units = p.rows * p.heads * p.ratio;
            const int64_t unit = split * units + row * p.heads * p.ratio + qh;
            float *dst = (float *)p.ws + unit * D + d;
            if (sum != 0.0f)
#pragma unroll
                for (int u = 0; u < N; ++u) dst[u] = o[u];
            if (d == 0) {
                float *ml = (float *)p.ws + units * p.splits * D + unit * 2;
                ml[0] = m;
                ml[1] = sum;
            }
        }
    }
}

// The parts of a split launch: a workgroup per row and query head.  Its lanes
// first share the parts' statistics out, then D/4 lanes by 1024/D of them take
// parts in turns; sums are in a fixed order.  (One group of lanes walking the
// parts in a chain waits for memory at every part: 102 us for 32 rows of 128
// parts.)
template <typename T, int D>
__device__ __forceinline__ void combine(const PhxKv4 &p) {
    constexpr int L = D / 4, G = 256 / L;
    __shared__ float factor[PHX_KV4_SPLITS];
    __shared__ float wave_m[4], wave_l[4];
    __shared__ phx_f4 sums[G][L];
    const int64_t heads = p.heads * p.ratio;
    const int64_t qh = blockIdx.x % heads, i = blockIdx.x / heads % p.max_q;
    const Seq s = kv4_seq(p, blockIdx.x / heads / p.max_q);
    const int64_t row = s.row0 + i;
    if (i >= s.count || row < 0 || row >= p.rows) return;
    const int64_t units = p.rows * heads, unit = row * heads + qh;
    const float *ml = (const float *)p.ws + units * p.splits * D;
    const int t = threadIdx.x;
    float m = KV4_NONE, l = 0.0f;
    if (t < p.splits) {
        const float2 w = *(const float2 *)(ml + (t * units + unit) * 2);
        l = w.y;
        if (l != 0.0f) m = w.x;
    }
    float top = m;
    for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    if ((t & 63) == 0) wave_m[t >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(wave_m[0], wave_m[1]), fmaxf(wave_m[2], wave_m[3]));
    // a part without keys has stored no sums: its factor of 0 skips them
    const float f = l != 0.0f ? __builtin_amdgcn_exp2f(m - top) : 0.0f;
    if (t < p.splits) factor[t] = f;
    float sum = f * l;
    for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
    if ((t & 63) == 0) wave_l[t >> 6] = sum;
    __syncthreads();
    const int g = t / L, lane = t % L;
    const float *part = (const float *)p.ws + unit * D + lane * 4;
    phx_f4 o = {0, 0, 0, 0};
#pragma unroll 4
    for (int x = g; x < p.splits; x += G) {
        const float w = factor[x];
        if (w == 0.0f) continue;
        const phx_f4 v = *(const phx_f4 *)(part + x * units * D);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(w, v[e], o[e]);
    }
    sums[g][lane] = o;
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int x = 1; x < G; ++x) o = o + sums[x][lane];
    const float out[4] = {o[0], o[1], o[2], o[3]};
    store<T, 4>((T *)p.y + row * p.ldy + qh * D + lane * 4, out,
                (wave_l[0] + wave_l[1]) + (wave_l[2] + wave_l[3]));
}

}  // namespace

#define ATTEND(T, D, suffix, NC, WAVES)                                                         \
    extern "C" __global__ __launch_bounds__(64 * KV4_WAVES, WAVES) void kv4_attend_##suffix##_c##NC( \
        PhxKv4 p) {                                                                             \
        attend<T, D, NC>(p);                                                                    \
    }
#define COMBINE(T, D, suffix)                                                                   \
    extern "C" __global__ __launch_bounds__(256) void kv4_combine_##suffix(PhxKv4 p) {          \
        combine<T, D>(p);                                                                       \
    }
ATTEND(_Float16, 64, f16_d64, 1, 2)
ATTEND(_Float16, 128, f16_d128, 1, 2)
ATTEND(float, 64, f32_d64, 1, 2)
ATTEND(float, 128, f32_d128, 1, 2)
ATTEND(_Float16, 64, f16_d64, 2, 2)
ATTEND(_Float16, 128, f16_d128, 2, 2)
ATTEND(float, 64, f32_d64, 2, 2)
ATTEND(float, 128, f32_d128, 2, 1)
ATTEND(_Float16, 64, f16_d64, 4, 1)
ATTEND(_Float16, 128, f16_d128, 4, 1)
COMBINE(_Float16, 64, f16_d64)
COMBINE(_Float16, 128, f16_d128)
COMBINE(float, 64, f32_d64)
COMBINE(float, 128, f32_d128)
