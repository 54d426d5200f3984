"""Every kernel of gemm_f8.hip by itself: dense, over groups of A's own rows and through
a list, with K of several rounds of the stage ring and of the scales (the rows' come
four blocks at a time, the weights' 64), starting at the first block or (few rows, blocks
in fours) at a workgroup's own.  test_f8_kernel_shapes.py says without a GPU that each
shape takes the kernel that it is listed under.

Codes of 1 and -1 and scales that are powers of two give results that are exact, in f16
too: multiples of 1/2 below 1024.  Every k counts in every one of them."""
import numpy as np
import pytest

import f8_model as f8
import test_gpu_gemm_f8 as gemm
from hip_graph import Graph

pytestmark = pytest.mark.gpu

NAN = 0x7F
# dense: (M, N, K); grouped: (M, experts, N, K)
KERNELS = {
    "f16_1x1_2x1_k4_s4": ([(1, 33, 8336), (1, 70, 4592)], [(7, 3, 33, 8336), (7, 3, 70, 4592)]),
    "f16_1x1_2x1_k4_s2": ([(1, 33, 1168), (5, 70, 1520)], [(7, 3, 33, 1168), (7, 3, 70, 1520)]),
    "f16_2x1_2x1_k4_s3": ([(513, 257, 1296), (513, 257, 8336), (33, 3000, 1520)],
                          [(400, 3, 300, 1296), (400, 9, 257, 1520)]),
    "f16_2x1_2x2_k2_s3": ([(513, 520, 1168), (513, 520, 8336), (63, 4099, 1520)],
                          [(1000, 3, 257, 1168), (257, 3, 1025, 1520)]),
    "f16_2x2_2x2_k2_s4": ([(1000, 520, 8336), (100, 4099, 4592)],
                          [(1000, 3, 520, 8336), (513, 3, 1025, 4592)]),
    "f16_2x2_2x2_k1_s4": ([(1000, 520, 1296), (1000, 1025, 8336), (100, 8200, 1520)],
                          [(1000, 3, 520, 1296), (513, 3, 2050, 1520)]),
    "f16_2x2_4x2_k1_s3": ([(1000, 2050, 1168), (2049, 1500, 8336), (130, 12000, 1520)],
                          [(3000, 3, 700, 1168), (700, 4, 3000, 1520)]),
    "f16_2x4_8x2_k1_s3": ([(2049, 2050, 1168), (2049, 2050, 8336)], [(4100, 3, 1025, 1168)]),
    "f16_2x4_8x4_k1_s2": ([(2049, 4099, 1168), (2049, 4099, 8336)], [(4100, 3, 2050, 1168)]),
    "f32_1x1_2x1_k4_s2": ([(1, 33, 1168), (513, 257, 8336), (5, 70, 1520)],
                          [(7, 3, 33, 1168), (7, 3, 70, 1520)]),
    "f32_1x1_2x1_k8_s3": ([(1, 33, 8336), (5, 70, 8688)], [(7, 3, 33, 8336), (7, 3, 70, 8688)]),
    "f32_2x1_2x2_k2_s3": ([(513, 520, 1168), (400, 1025, 8336), (65, 8200, 1520)],
                          [(1000, 3, 257, 1168), (257, 3, 1500, 1520)]),
    "f32_1x2_4x2_k4_s2": ([(1000, 520, 1296), (1000, 520, 8336), (100, 4099, 1520)],
                          [(1000, 3, 520, 1296), (513, 3, 1025, 1520)]),
    "f32_2x2_2x2_k1_s4": ([(1000, 1025, 1168), (1000, 1025, 8336), (100, 8200, 1520)],
                          [(1500, 3, 700, 1168), (513, 3, 2050, 1520)]),
    "f32_2x2_4x2_k1_s3": ([(1000, 2050, 1168), (1000, 2050, 8336), (130, 12000, 1520)],
                          [(3000, 3, 700, 1168), (700, 4, 3000, 1520)]),
    "f32_2x2_4x4_k1_s2": ([(2049, 2050, 1168), (2049, 2050, 8336)], [(4100, 3, 1025, 1168)]),
}
DENSE = [(k, s) for k, (dense, _) in KERNELS.items() for s in dense]
GROUPED = [(k, s) for k, (_, grouped) in KERNELS.items() for s in grouped]
FIRST = [(k, dense[0]) for k, (dense, _) in KERNELS.items()]
FIRST_GROUPED = [(k, grouped[0]) for k, (_, grouped) in KERNELS.items()]


def _bits(kernel):
    return int(kernel[1:3])


class Signs:
    """Codes [lead, width] of 1 and -1 and their scales on the device, rows ld and lds
    apart, NaN behind every row and at the end."""

    def __init__(self, px, rng, lead, width, scales, ld, lds):
        self.codes = rng.integers(0, 2, (lead, width), dtype=np.uint8) << 7 | np.uint8(0x38)
        self.scales, self.ld, self.lds = scales.astype(np.float32), ld, lds
        c, s = np.full((lead, ld), NAN, np.uint8), np.full((scales.shape[0], lds), np.nan, np.float32)
        c[:, :width], s[:, :scales.shape[1]] = self.codes, scales
        self.c = px.DeviceBuffer.from_array(np.concatenate([c.ravel(), np.full(4096, NAN, np.uint8)]))
        self.s = px.DeviceBuffer.from_array(np.concatenate([s.ravel(), np.full(64, np.nan, np.float32)]))

    def signs(self, lo=0, hi=None):
        return np.where(self.codes[lo:hi] >> 7, np.float32(-1), np.float32(1))


class Rows(Signs):
    def __init__(self, px, rng, M, K):
        kb = -(-K // 128)
        super().__init__(px, rng, M, K, 2.0 ** rng.integers(0, 2, (M, kb)), K + 16, -(-kb // 4) * 4 + 4)
        self.rows = px.F8Rows(self.c.ptr, self.s.ptr, M, K, self.ld, self.lds)

    def values(self):
        return self.signs() * np.repeat(self.scales, 128, 1)[:, :self.codes.shape[1]]


class Weights(Signs):
    def __init__(self, px, rng, E, N, K):
        self.N, self.K, self.nb, kb = N, K, -(-N // 128), -(-K // 128)
        super().__init__(px, rng, E * N, K, 2.0 ** rng.integers(-1, 1, (E * self.nb, kb)), K, kb)
        self.weights = px.F8Weights(self.c.ptr, self.s.ptr, E, N, K)

    def values(self, e):
        s = self.scales[e * self.nb:(e + 1) * self.nb]
        s = np.repeat(np.repeat(s, 128, 0)[:self.N], 128, 1)[:, :self.K]
        return self.signs(e * self.N, (e + 1) * self.N) * s


def _exact(want):
    assert np.abs(want).max() <= 1024  # in halves: what f16 has
    return want


@pytest.mark.parametrize("kernel,shape", DENSE)
def test_dense(px_gpu, stream, kernel, shape):
    M, N, K = shape
    rng = np.random.default_rng(M + N + K)
    a, w = Rows(px_gpu, rng, M, K), Weights(px_gpu, rng, 1, N, K)
    want = _exact(a.values() @ w.values(0).T)
    got = gemm._run(px_gpu, stream, _bits(kernel), a, w, M, ldc=N + 3)
    assert np.array_equal(got.astype(np.float32), want)


@pytest.mark.parametrize("kernel,shape", FIRST)
def test_nan_stays_in_its_row_and_column(px_gpu, stream, kernel, shape):
    px, (M, N, K) = px_gpu, shape
    rng = np.random.default_rng(M + N)
    a, w = Rows(px, rng, M, K), Weights(px, rng, 1, N, K)
    want = _exact(a.values() @ w.values(0).T)
    bad = np.zeros((M, N), bool)
    if M > 4:
        codes, scales = (b.download(t, b.nbytes // t().itemsize)
                         for b, t in ((a.c, np.uint8), (a.s, np.float32)))
        rows = [M // 7, M // 2, M - 1]
        codes[rows[0] * a.ld + 9], codes[rows[1] * a.ld + K - 1] = 0x7F, 0xFF
        scales[rows[2] * a.lds + K // 128] = np.nan
        a.c.upload(codes)
        a.s.upload(scales)
        bad[rows] = True
    codes = w.c.download(np.uint8, w.c.nbytes)
    for n, k in ((N // 3, 200), (N - 2, K - 1)):
        codes[n * K + k] = 0xFF
        bad[:, n] = True
    w.c.upload(codes)
    if N > 256:  # a block of weights' scale: its 128 columns
        scales = w.s.download(np.float32, w.s.nbytes // 4)
        scales[w.scales.shape[1] + 5] = np.nan
        w.s.upload(scales)
        bad[:, 128:256] = True
    got = gemm._run(px, stream, _bits(kernel), a, w, M)
    assert np.isnan(got[bad]).all()
    assert np.array_equal(got[~bad].astype(np.float32), want[~bad])


def _routes(rng, M, E, rows):
    """Starts as they may be handed over (one descends, one leaves 0 .. M where there is
    no row left out), as they count, the rows in no group, and a list with entries that
    are no rows."""
    lead, tail = (0, 0) if M < 20 else (3, 5)
    edges = np.sort(rng.integers(lead, M - tail + 1, E - 1))
    starts = np.concatenate([[lead], edges, [M - tail]])
    starts[1] = min(starts[1] + M // 9, M - tail)
    starts[2] = max(starts[1] - 2, 0)
    if not lead:
        starts[0], starts[-1] = -7, M + 9
    counts = np.maximum.accumulate(np.clip(starts, 0, M))
    order = rng.integers(0, rows, M)
    order[rng.integers(0, M, 1 + M // 50)] = rng.choice([-1, rows, 1 << 30, -(1 << 31)])
    return starts, counts, np.r_[0:counts[0], counts[-1]:M], order


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("kernel,shape", GROUPED)
def test_grouped(px_gpu, stream, kernel, shape, listed):
    M, E, N, K = shape
    rng = np.random.default_rng(M + N + K)
    rows = M // 2 + 1 if listed else M
    a, w = Rows(px_gpu, rng, rows, K), Weights(px_gpu, rng, E, N, K)
    starts, counts, left, order = _routes(rng, M, E, rows)
    x = a.values()
    if listed:
        x = np.where(((order >= 0) & (order < rows))[:, None], x[np.clip(order, 0, rows - 1)], 0)
    got = gemm._run(px_gpu, stream, _bits(kernel), a, w, M, starts, order if listed else None,
                    ldc=N + 5, left=left)
    for e, (b, end) in enumerate(zip(counts, counts[1:])):
        want = x[b:end] @ w.values(e).T
        if b < end:
            assert np.array_equal(got[b:end].astype(np.float32), _exact(want))


@pytest.mark.parametrize("kernel,shape", FIRST)
def test_normal_inputs_onto_c(px_gpu, stream, kernel, shape):
    M, N, K = shape
    rng = np.random.default_rng(N)
    bits = _bits(kernel)
    t = np.float16 if bits == 16 else np.float32
    a, w = gemm._normal(px_gpu, rng, M, N, K, pad=1)
    product = a.values @ w.values[0].T
    got = gemm._run(px_gpu, stream, bits, a, w, M)
    assert (np.abs(got - product) <= gemm._bound(product, a.values, w.values[0], t)).all()
    c = (rng.standard_normal((M, N)) * np.abs(product).max()).clip(-6e4, 6e4).astype(t)
    want = 0.5 * product - 1.5 * c.astype(np.float64)
    got = gemm._run(px_gpu, stream, bits, a, w, M, alpha=0.5, beta=-1.5, c=c, ldc=N + 1)
    fits = np.abs(want) < (65000 if bits == 16 else np.inf)
    bound = gemm._bound(want, a.values, w.values[0], t, 0.5, 1.5 * np.abs(c.astype(np.float64)))
    assert (np.abs(got - want) <= bound)[fits].all()


@pytest.mark.parametrize("kernel,shape", FIRST_GROUPED)
def test_grouped_normal_inputs_onto_c(px_gpu, stream, kernel, shape):
    M, E, N, K = shape
    rng = np.random.default_rng(K)
    bits = _bits(kernel)
    t = np.float16 if bits == 16 else np.float32
    a, w = gemm._normal(px_gpu, rng, 70, N, K, E)
    starts, counts, left, order = _routes(rng, M, E, 70)
    c = rng.standard_normal((M, N)).astype(t)
    got = gemm._run(px_gpu, stream, bits, a, w, M, starts, order, 2.0, 1.0, c, left=left)
    for e, (b, end) in enumerate(zip(counts, counts[1:])):
        rows = gemm._rows_in(a, order, b, end)
        want = 2 * (rows @ w.values[e].T) + c[b:end].astype(np.float64)
        bound = gemm._bound(want, rows, w.values[e], t, 2.0, np.abs(c[b:end].astype(np.float64)))
        assert (np.abs(got[b:end] - want) <= bound).all()


@pytest.mark.parametrize("kernel", ["f16_1x1_2x1_k4_s4", "f16_2x1_2x2_k2_s3", "f16_2x2_4x2_k1_s3",
                                    "f16_2x4_8x4_k1_s2", "f32_1x1_2x1_k8_s3", "f32_2x2_4x4_k1_s2"])
def test_captured_and_replayed(px_gpu, kernel):
    # rows, starts and lists change between the replays, C is accumulated onto
    px = px_gpu
    dense, grouped = KERNELS[kernel]
    (M, N, K), (R, E, GN, GK) = dense[0], grouped[0]
    dt, t = gemm._t(px, _bits(kernel))
    rng = np.random.default_rng(1)
    s = px.Stream()
    a, w = Rows(px, rng, M, K), Weights(px, rng, 1, N, K)
    ga, gw = Rows(px, rng, R, GK), Weights(px, rng, E, GN, GK)
    c, gc = px.DeviceBuffer(M * N * t().itemsize), px.DeviceBuffer(R * GN * t().itemsize)
    ds, do = px.DeviceBuffer(4 * (E + 1)), px.DeviceBuffer(4 * R)

    def step():
        px.launch_gemm_f8(s, a.rows, w.weights, dt, c, 1.0, 0.5)
        px.launch_gemm_f8_grouped(s, ga.rows, gw.weights, ds, do, R, dt, gc, 1.0, 0.5)

    def inputs():
        starts, _, _, order = _routes(rng, R, E, R)
        ds.upload(starts.astype(np.int32))
        do.upload(order.astype(np.int32))
        for x in (a, ga):
            codes = x.c.download(np.uint8, x.c.nbytes)
            codes[codes != NAN] ^= 0x80 * (rng.random((codes != NAN).sum()) < 0.5).astype(np.uint8)
            x.c.upload(codes)

    def zero():
        for b in (c, gc):
            b.upload(np.full(b.nbytes // t().itemsize, 2, t))
    inputs()
    zero()
    step()
    s.synchronize()
    g = Graph(s, step)
    for _ in range(4):
        inputs()
        zero()
        step()
        s.synchronize()
        want = [b.download(t, b.nbytes // t().itemsize).copy() for b in (c, gc)]
        zero()
        g.replay()
        s.synchronize()
        for b, x in zip((c, gc), want):
            assert np.array_equal(b.download(t, b.nbytes // t().itemsize), x)
    g.destroy()
    s.destroy()


# ---------------------------------------------------------------- f16, where only f32 was run
def test_every_code(px_gpu, stream):
    # all finite e4m3 codes are f16 numbers
    codes = np.zeros((254, 128), np.uint8)
    finite = [c for c in range(256) if c & 127 != 127]
    codes[np.arange(254), np.arange(254) % 128] = finite
    one = int(f8.codes_of(1.0))
    a = gemm.Rows(px_gpu, codes, np.ones((254, 1)))
    w = gemm.Weights(px_gpu, np.full((1, 20, 128), one, np.uint8), np.ones((1, 1, 1)))
    got = gemm._run(px_gpu, stream, 16, a, w, 254)
    assert np.array_equal(got, np.repeat(f8.VALUES[finite][:, None], 20, 1))
    a = gemm.Rows(px_gpu, np.full((3, 128), one, np.uint8), np.ones((3, 1)))
    w = gemm.Weights(px_gpu, codes[None], np.ones((1, 2, 1)))
    got = gemm._run(px_gpu, stream, 16, a, w, 3)
    assert np.array_equal(got, np.repeat(f8.VALUES[finite][None], 3, 0))


@pytest.mark.parametrize("M,N", [(9, 140), (300, 4200)])
def test_scales_of_every_size(px_gpu, stream, M, N):
    # f16's smallest and largest results, one that is infinite, zero scales, and scales
    # whose product alone is in f32's range
    px, K = px_gpu, 512
    one = int(f8.codes_of(1.0))
    e = np.array([-40, -31, -30, -20, -3, 0, 5, 8, 9])[np.arange(M) % 9]
    shift = np.where(np.arange(-(-N // 128)) % 3 == 1, 0, 100)
    sa, sw = 2.0 ** (e - 100.0), 2.0 ** (shift - 3.0)
    sw[shift == 0] = 0
    a = gemm.Rows(px, np.full((M, K), one, np.uint8), np.repeat(sa[:, None], 4, 1))
    w = gemm.Weights(px, np.full((1, N, K), one, np.uint8), np.repeat(sw[:, None], 4, 1)[None])
    got = gemm._run(px, stream, 16, a, w, M)
    with np.errstate(over="ignore"):
        want = (a.values @ w.values[0].T).astype(np.float16)
    assert np.array_equal(got, want)
    got = gemm._run(px, stream, 16, a, w, M, alpha=2.0)  # 512 * 2^9 / 8 * 2: infinite
    with np.errstate(over="ignore"):
        want = (2 * (a.values @ w.values[0].T)).astype(np.float16)
    assert np.array_equal(got, want) and np.isinf(got).any()


def test_a_list_over_no_rows_at_all(px_gpu, stream):
    px = px_gpu
    rng = np.random.default_rng(4)
    w = Weights(px, rng, 3, 70, 144)
    a = type("Nothing", (), {"rows": px.F8Rows(0, 0, 0, 144, 160)})
    c = rng.standard_normal((9, 70)).astype(np.float16)
    got = gemm._run(px, stream, 16, a, w, 9, [0, 4, 4, 9], rng.integers(-3, 3, 9), 1.0, 2.0, c)
    assert np.array_equal(got, 2 * c)


@pytest.mark.parametrize("E,M", [(3000, 40), (65535, 3), (65, 400), (128, 129)])
def test_many_experts(px_gpu, stream, E, M):
    rng = np.random.default_rng(E)
    a, w = Rows(px_gpu, rng, M, 32), Weights(px_gpu, rng, E, 3, 32)
    counts = rng.multinomial(M, np.ones(E) / E)
    starts = np.concatenate([[0], np.cumsum(counts)])
    got = gemm._run(px_gpu, stream, 16, a, w, M, starts)
    x = a.values()
    for e in np.flatnonzero(counts):
        b, end = starts[e], starts[e + 1]
        assert np.array_equal(got[b:end].astype(np.float32), x[b:end] @ w.values(e).T)


@pytest.mark.parametrize("M,N,K", [(40, 300, 128), (300, 520, 1040), (2049, 2100, 272)])
@pytest.mark.parametrize("cancel", [False, True])
@pytest.mark.parametrize("bits", [16, 32])
def test_products_of_every_size(px_gpu, stream, bits, cancel, M, N, K):
    # codes of every size next to each other; cancel: the large products come in pairs
    # that cancel, so that what a result has left shows what the sums lost
    px = px_gpu
    rng = np.random.default_rng(K)
    t = np.float16 if bits == 16 else np.float32
    finite = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    a, w = rng.choice(finite, (M, K)), rng.choice(finite, (1, N, K))
    if cancel:
        a[:, 1::2], w[..., 1::2] = a[:, ::2], w[..., ::2] ^ 0x80
        a[:, 3::8] = rng.choice(finite, a[:, 3::8].shape)
    kb = -(-K // 128)
    a = gemm.Rows(px, a, np.full((M, kb), 2.0 ** -4))
    w = gemm.Weights(px, w, np.full((1, -(-N // 128), kb), 2.0 ** -6))
    want = a.values @ w.values[0].T
    got = gemm._run(px, stream, bits, a, w, M)
    fits = np.abs(want) < (65000 if bits == 16 else np.inf)
    assert (np.abs(got - want) <= gemm._bound(want, a.values, w.values[0], t))[fits].all()
