"""phx_gemm_f8 and phx_gemm_f8_grouped against 64 bits.  With small whole numbers
and scales that are powers of two every product and partial sum is exact, so the
result has to be the exact one: any wrong index, block or mask shows.  With normal
inputs the bound is the arithmetic's: f32 sums of K products, one rounding of the
output.  Bytes that are no part of a row or a weight are codes of NaN, scales that
are none are NaN."""
import numpy as np
import pytest

import f8_model as f8
from hip_graph import Graph

pytestmark = pytest.mark.gpu

GUARD = 64
NAN = 0x7F


def _t(px, bits):
    return (px.F16, np.float16) if bits == 16 else (px.F32, np.float32)


class Rows:
    """8-bit rows on the device, with strides and NaN behind every row."""

    def __init__(self, px, codes, scales, pad=0):
        M, K = codes.shape
        kb = scales.shape[1]
        ld, lds = K + 16 * pad, -(-kb // 4) * 4 + 4 * pad
        c, s = np.full((M, ld), NAN, np.uint8), np.full((M, lds), np.nan, np.float32)
        c[:, :K], s[:, :kb] = codes, scales
        self.c = px.DeviceBuffer.from_array(np.concatenate([c.ravel(), np.full(4096, NAN, np.uint8)]))
        self.s = px.DeviceBuffer.from_array(s)
        self.rows = px.F8Rows(self.c.ptr, self.s.ptr, M, K, ld if pad else 0, lds if pad else 0)
        self.values = f8.row_values(codes, scales)


class Weights:
    def __init__(self, px, codes, scales):
        E, N, K = codes.shape
        self.c = px.DeviceBuffer.from_array(
            np.concatenate([codes.ravel(), np.full(4096, NAN, np.uint8)]))
        self.s = px.DeviceBuffer.from_array(
            np.concatenate([scales.astype(np.float32).ravel(), np.full(64, np.nan, np.float32)]))
        self.weights = px.F8Weights(self.c.ptr, self.s.ptr, E, N, K)
        self.values = f8.weight_values(codes, scales)


def _whole(px, rng, M, N, K, E=1, pad=0, bits=32):
    """Whole numbers of up to 8 and scales of 1/2 .. 2: sums below 2^24 quarters; for
    f16, a few elements a row of up to 2 and scales of up to 1: below 2^11 quarters."""
    few = min(1.0, 2000 / K)

    def draw(*shape):
        v = rng.integers(-8, 9, shape) * (rng.random(shape) < few)
        if bits == 16:  # |v| <= 2 in each row, 16 of them in a row of A
            v = np.clip(v, -2, 2)
            if len(shape) == 2:
                keep = np.zeros(shape, bool)
                for m in range(shape[0]):
                    keep[m, rng.choice(K, min(K, 16), replace=False)] = True
                v = v * keep
        return f8.codes_of(v)
    if bits == 16:
        kb, nb = -(-K // 128), -(-N // 128)
        a = Rows(px, draw(M, K), 2.0 ** rng.integers(-1, 1, (M, kb)), pad)
        return a, Weights(px, draw(E, N, K), 2.0 ** rng.integers(-1, 1, (E, nb, kb)))
    kb, nb = -(-K // 128), -(-N // 128)
    a = Rows(px, draw(M, K), 2.0 ** rng.integers(-1, 2, (M, kb)), pad)
    w = Weights(px, draw(E, N, K), 2.0 ** rng.integers(-1, 1, (E, nb, kb)))
    return a, w


def _normal(px, rng, M, N, K, E=1, pad=0):
    def draw(lead, width):
        x = rng.standard_normal((lead, width)) * 10.0 ** rng.uniform(-2, 2, (lead, 1))
        q, a = f8.quotients(x)
        return f8.codes_of(q), (a / 448).astype(np.float32)
    kb, nb = -(-K // 128), -(-N // 128)
    a = Rows(px, *draw(M, K), pad)
    codes, _ = draw(E * N, K)
    w = Weights(px, codes.reshape(E, N, K), (rng.random((E, nb, kb)) * 1e-3 + 1e-5).astype(np.float32))
    return a, w


def _run(px, stream, bits, a, w, M, starts=None, order=None, alpha=1.0, beta=0.0, c=None, ldc=0,
         left=None):
    """C's rows; what lies between and around them, and the rows `left`, has to stay."""
    dt, t = _t(px, bits)
    N = w.weights.n
    ld = ldc or N
    out = np.full(GUARD + M * ld + GUARD, 77, t)
    view = out[GUARD:GUARD + M * ld].reshape(M, ld)
    if c is not None:
        view[:, :N] = c
    elif beta == 0.0:
        view[:, :N] = np.nan  # not read
    buf = px.DeviceBuffer.from_array(out)
    at = buf.ptr + GUARD * out.itemsize
    if starts is None:
        px.launch_gemm_f8(stream, a.rows, w.weights, dt, at, alpha, beta, ldc)
    else:
        ds = px.DeviceBuffer.from_array(np.asarray(starts, np.int32))
        do = px.DeviceBuffer.from_array(np.asarray(order, np.int32)) if order is not None else 0
        px.launch_gemm_f8_grouped(stream, a.rows, w.weights, ds, do, M, dt, at, alpha, beta, ldc)
    stream.synchronize()
    got = buf.download(t, out.shape)
    kept = np.ones(out.shape, bool)
    inside = kept[GUARD:GUARD + M * ld].reshape(M, ld)
    inside[:, :N] = False
    if left is not None:
        inside[left] = True
    assert np.array_equal(got[kept], out[kept], equal_nan=True), "stored outside C"
    return got[GUARD:GUARD + M * ld].reshape(M, ld)[:, :N]


def _most(a, w):
    """For each result the sum, over groups of eight k, of the largest product that
    the group can have."""
    def largest(x):
        x = np.pad(np.abs(x), ((0, 0), (0, -x.shape[1] % 8)))
        return x.reshape(x.shape[0], x.shape[1] // 8, 8).max(-1)
    return largest(a) @ largest(w).T


def _bound(want, a, w, t, alpha=1.0, extra=0.0):
    """Half a step of the output, and f32's of K products, their scales and sums,
    alpha and beta; for f16 of eight neighbouring products seven lose less than
    2^-13 of the largest each."""
    half, K = np.finfo(t).eps / 2, a.shape[1]
    inner = ((K + 8) * (np.abs(a) @ np.abs(w).T) * abs(alpha) + 2 * extra + np.abs(want)) * 2.0 ** -24
    if t == np.float16:
        inner = inner + 7 * 2.0 ** -13 * _most(a, w) * abs(alpha)
    tiny = 2.0 ** -25 if t == np.float16 else 2.0 ** -149
    return (np.abs(want) + inner) * half + inner + tiny


SHAPES = [(1, 1, 16), (1, 16, 128), (2, 17, 144), (3, 5, 32), (15, 33, 112), (16, 16, 256),
          (17, 40, 400), (33, 100, 80), (64, 15, 528), (48, 257, 1040), (1, 1000, 4144), (4, 64, 8192),
          (65, 130, 2064), (5, 4099, 64), (1, 31, 16384), (127, 129, 272), (128, 128, 1024),
          (129, 300, 640), (200, 1030, 384), (256, 256, 512), (300, 520, 1040), (257, 255, 2048),
          (513, 700, 128), (1000, 1000, 16), (1030, 2050, 656), (5, 700, 2048), (64, 300, 1024), (100, 500, 512),
          (33, 9000, 3584), (256, 260, 1536), (20, 500, 4608), (7, 100, 20480)]


# more tiles of every kind than the GPU runs at a time, last ones short
LARGE = [(2049, 4111, 272), (4100, 4090, 144), (1, 16500, 528), (40, 16390, 272), (700, 9000, 144),
         (8200, 300, 400), (1, 12000, 4144), (33, 3000, 4144), (33, 6000, 4144), (100, 4000, 4144),
         (17, 16000, 2064), (300, 16000, 528)]


@pytest.mark.parametrize("M,N,K", SHAPES + LARGE)
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("pad", [0, 1])
def test_whole_numbers_are_exact(px_gpu, stream, bits, M, N, K, pad):
    rng = np.random.default_rng(M * 7 + N * 3 + K)
    a, w = _whole(px_gpu, rng, M, N, K, pad=pad, bits=bits)
    want = a.values @ w.values[0].T
    got = _run(px_gpu, stream, bits, a, w, M, ldc=N + 3 * pad)
    assert np.array_equal(got.astype(np.float64), want)


@pytest.mark.parametrize("M,N,K", [(1, 48, 4096), (5, 1000, 4144), (16, 333, 528), (64, 100, 2048),
                                   (23, 18, 8192), (130, 140, 2064), (300, 520, 1040), (700, 256, 4096),
                                   (40, 2100, 528), (2049, 1025, 400)])
@pytest.mark.parametrize("bits", [16, 32])
def test_normal_inputs(px_gpu, stream, bits, M, N, K):
    rng = np.random.default_rng(K + N)
    _, t = _t(px_gpu, bits)
    a, w = _normal(px_gpu, rng, M, N, K, pad=1)
    want = a.values @ w.values[0].T
    got = _run(px_gpu, stream, bits, a, w, M, ldc=N + 3)
    assert (np.abs(got - want) <= _bound(want, a.values, w.values[0], t)).all()
    # f16: all in all no further off than the rounding of each result may be
    off = np.linalg.norm(got - want, axis=1) / np.linalg.norm(want, axis=1)
    assert (off <= np.finfo(t).eps / 2 * (1 if bits == 16 else 8)).all()


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("M,N,K", [(6, 50, 640), (260, 300, 272), (70, 514, 2064)])
@pytest.mark.parametrize("odd", [0, 1])
def test_alpha_and_beta(px_gpu, stream, bits, M, N, K, odd):
    rng = np.random.default_rng(3)
    _, t = _t(px_gpu, bits)
    a, w = _normal(px_gpu, rng, M, N, K)
    want = a.values @ w.values[0].T
    c = (rng.standard_normal((M, N)) * np.abs(want).max()).clip(-6e4, 6e4).astype(t)
    want = 0.5 * want - 1.5 * c.astype(np.float64)
    got = _run(px_gpu, stream, bits, a, w, M, alpha=0.5, beta=-1.5, c=c, ldc=N + odd)
    fits = np.abs(want) < (65000 if bits == 16 else np.inf)
    bound = _bound(want, a.values, w.values[0], t, 0.5, 1.5 * np.abs(c.astype(np.float64)))
    assert (np.abs(got - want) <= bound)[fits].all()
    # alpha 0 and a C of NaN: not read with beta 0
    assert (_run(px_gpu, stream, bits, a, w, M, alpha=0.0, beta=0.0) == 0).all()


def test_every_code(px_gpu, stream):
    # a row of one code each against weights of 1: the code's value
    codes = np.zeros((254, 128), np.uint8)
    finite = [c for c in range(256) if c & 127 != 127]
    codes[np.arange(254), np.arange(254) % 128] = finite
    a = Rows(px_gpu, codes, np.ones((254, 1)))
    w = Weights(px_gpu, np.full((1, 20, 128), f8.codes_of(1.0), np.uint8), np.ones((1, 1, 1)))
    got = _run(px_gpu, stream, 32, a, w, 254)
    assert np.array_equal(got, np.repeat(f8.VALUES[finite][:, None], 20, 1))
    # and of one weight each
    a = Rows(px_gpu, np.full((3, 128), f8.codes_of(1.0), np.uint8), np.ones((3, 1)))
    w = Weights(px_gpu, codes[None], np.ones((1, 2, 1)))
    got = _run(px_gpu, stream, 32, a, w, 3)
    assert np.array_equal(got, np.repeat(f8.VALUES[finite][None], 3, 0))


@pytest.mark.parametrize("M,N,K", [(7, 40, 272), (300, 300, 272)])
def test_nan_stays_in_its_row_and_column(px_gpu, stream, M, N, K):
    rng = np.random.default_rng(5)
    a, w = _whole(px_gpu, rng, M, N, K)
    clean = _run(px_gpu, stream, 32, a, w, M)
    codes = a.c.download(np.uint8, M * K).copy()
    codes[2 * K + 9], codes[4 * K + K - 1] = 0x7F, 0xFF
    a.c.upload(codes)
    scales = a.s.download(np.float32, (M, a.s.nbytes // 4 // M)).copy()
    scales[5, 1] = np.nan
    a.s.upload(scales)
    wc = w.c.download(np.uint8, N * K).copy()
    wc[33 * K + 200] = 0x7F
    w.c.upload(wc)
    got = _run(px_gpu, stream, 32, a, w, M)
    bad = np.zeros((M, N), bool)
    bad[[2, 4, 5]] = True
    bad[:, 33] = True
    assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], clean[~bad])


def test_scales_of_every_size(px_gpu, stream):
    # tiny, zero and huge scales of rows meet those of weights in f32
    px = px_gpu
    M, N, K = 9, 140, 512
    one = f8.codes_of(1.0)
    sa = np.array([2.0 ** e for e in (-140, -126, -100, -10, 0, 20, 60, 100, 120)])[:, None]
    a = Rows(px, np.full((M, K), one, np.uint8), np.repeat(sa, 4, 1))
    sw = np.array([[2.0 ** -3] * 4, [0.0] * 4])
    w = Weights(px, np.full((1, N, K), one, np.uint8), sw[None])
    got = _run(px, stream, 32, a, w, M)
    assert np.array_equal(got.astype(np.float64), a.values @ w.values[0].T)


# ---------------------------------------------------------------- grouped
def _groups(rng, E, M, idle):
    live = np.sort(rng.choice(E, E - idle, replace=False))
    edges = np.sort(rng.integers(0, M + 1, live.size - 1))
    counts = np.zeros(E, np.int64)
    counts[live] = np.diff(np.concatenate([[0], edges, [M]]))
    return np.concatenate([[0], np.cumsum(counts)])


def _rows_in(a, order, b, end):
    """A's rows that rows b .. end of C take: zeros for an entry that is none."""
    if order is None:
        return a.values[b:end]
    i = np.asarray(order[b:end], np.int64)
    return np.where(((i >= 0) & (i < len(a.values)))[:, None],
                    a.values[np.clip(i, 0, len(a.values) - 1)], 0)


def _want(a, w, starts, order, M):
    out = np.zeros((M, w.weights.n))
    for e in range(w.weights.experts):
        b, end = starts[e], starts[e + 1]
        out[b:end] = _rows_in(a, order, b, end) @ w.values[e].T
    return out


GROUPED = [(1, 1, 1, 16, 0), (5, 3, 17, 144, 1), (40, 7, 100, 272, 2), (16, 32, 260, 1040, 18),
           (300, 4, 130, 400, 0), (1000, 6, 257, 256, 1), (700, 64, 140, 128, 30), (3, 200, 33, 64, 190),
           (129, 130, 16, 528, 3), (2000, 3, 300, 272, 1), (60, 2, 2050, 400, 0), (50, 9, 300, 1024, 3), (200, 3, 500, 512, 0),
           (9, 4, 5000, 2048, 1)]


@pytest.mark.parametrize("M,E,N,K,idle", GROUPED)
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("listed", [False, True])
def test_grouped_whole_numbers_are_exact(px_gpu, stream, bits, M, E, N, K, idle, listed):
    rng = np.random.default_rng(M + E * 3 + N)
    src = max(1, M // 2) if listed else M
    a, w = _whole(px_gpu, rng, src, N, K, E, pad=listed, bits=bits)
    starts = _groups(rng, E, M, idle)
    order = rng.integers(0, src, M) if listed else None
    want = _want(a, w, starts, order, M)
    got = _run(px_gpu, stream, bits, a, w, M, starts, order, ldc=N + 5)
    assert np.array_equal(got.astype(np.float64), want)


@pytest.mark.parametrize("each,E", [(1, 9), (17, 9), (33, 5), (65, 40), (129, 5), (257, 5), (257, 30)])
@pytest.mark.parametrize("bits", [16, 32])
def test_groups_of_one_row_more_than_whole_tiles(px_gpu, stream, bits, each, E):
    # as many tiles as M rows of E groups can have
    rng = np.random.default_rng(each)
    M = each * E
    a, w = _whole(px_gpu, rng, M, 270, 144, E, bits=bits)
    starts = np.arange(E + 1) * each
    got = _run(px_gpu, stream, bits, a, w, M, starts)
    assert np.array_equal(got.astype(np.float64), _want(a, w, starts, None, M))


@pytest.mark.parametrize("M,E,N,K,idle", [(50, 9, 300, 1040, 3), (1500, 8, 520, 400, 1)])
@pytest.mark.parametrize("bits", [16, 32])
def test_grouped_normal_inputs_onto_c(px_gpu, stream, bits, M, E, N, K, idle):
    rng = np.random.default_rng(8)
    _, t = _t(px_gpu, bits)
    a, w = _normal(px_gpu, rng, 70, N, K, E)
    starts, order = _groups(rng, E, M, idle), rng.integers(0, 70, M)
    want = _want(a, w, starts, order, M)
    c = rng.standard_normal((M, N)).astype(t)
    got = _run(px_gpu, stream, bits, a, w, M, starts, order, 2.0, 1.0, c)
    want = 2 * want + c.astype(np.float64)
    for e in range(E):
        b, end = starts[e], starts[e + 1]
        bound = _bound(want[b:end], _rows_in(a, order, b, end), w.values[e], t, 2.0,
                       np.abs(c[b:end].astype(np.float64)))
        assert (np.abs(got[b:end] - want[b:end]) <= bound).all()


@pytest.mark.parametrize("M,K", [(60, 272), (700, 128)])
def test_rows_outside_every_group_are_left(px_gpu, stream, M, K):
    rng = np.random.default_rng(1)
    a, w = _whole(px_gpu, rng, M, 140, K, 4)
    starts = np.array([5, 5, 20, 20, M - 11])
    left = np.r_[0:5, M - 11:M]
    got = _run(px_gpu, stream, 32, a, w, M, starts, left=left)
    want = _want(a, w, starts, None, M)
    keep = np.setdiff1d(np.arange(M), left)
    assert np.array_equal(got[keep], want[keep])
    # no group has a row
    _run(px_gpu, stream, 32, a, w, M, np.zeros(5), left=np.arange(M))


@pytest.mark.parametrize("M,K,N", [(60, 272, 140), (700, 128, 300)])
def test_starts_and_lists_that_are_wrong(px_gpu, stream, M, K, N):
    # starts that descend or leave 0 .. M, entries that are no rows of A: nothing is
    # read or written outside, and what the header says comes out
    rng = np.random.default_rng(2)
    a, w = _whole(px_gpu, rng, 30, N, K, 6)
    order = rng.integers(0, 30, M)
    order[[0, 7, 33]], order[[2, 50]], order[M - 1] = -1, 30, 1 << 30
    starts = np.array([-5, 9, 4, 40, -2147483648, 2147483647, M + 9])
    got = _run(px_gpu, stream, 32, a, w, M, starts, order)
    ascending = np.maximum.accumulate(np.clip(starts, 0, M))
    want = _want(a, w, ascending, order, M)
    assert np.array_equal(got, want)


def test_a_list_over_no_rows_at_all(px_gpu, stream):
    # every entry is no row: zeros, on top of C where beta says so
    px = px_gpu
    rng = np.random.default_rng(4)
    _, w = _whole(px, rng, 1, 70, 144, 3)
    a = type("Nothing", (), {"rows": px.F8Rows(0, 0, 0, 144, 160)})
    c = rng.standard_normal((9, 70)).astype(np.float32)
    got = _run(px, stream, 32, a, w, 9, [0, 4, 4, 9], rng.integers(-3, 3, 9), 1.0, 2.0, c)
    assert np.array_equal(got, 2 * c)


@pytest.mark.parametrize("E,M", [(3000, 40), (65535, 3), (65, 400), (64, 64), (128, 129)])
def test_many_experts(px_gpu, stream, E, M):
    rng = np.random.default_rng(E)
    a, w = _whole(px_gpu, rng, M, 3, 32, E)
    counts = rng.multinomial(M, np.ones(E) / E)
    starts = np.concatenate([[0], np.cumsum(counts)])
    got = _run(px_gpu, stream, 32, a, w, M, starts)
    want = np.zeros((M, 3))
    for e in np.flatnonzero(counts):
        want[starts[e]:starts[e + 1]] = a.values[starts[e]:starts[e + 1]] @ w.values[e].T
    assert np.array_equal(got, want)


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("M,N,K", [(2, 20, 1 << 22), (300000, 3, 16), (1, 200000, 48), (70000, 40, 144)])
def test_the_longest(px_gpu, stream, bits, M, N, K):
    rng = np.random.default_rng(K)
    _, t = _t(px_gpu, bits)
    a, w = _whole(px_gpu, rng, M, N, K, bits=bits if M < 100 else 32)
    want = a.values @ w.values[0].T
    got = _run(px_gpu, stream, bits, a, w, M)
    assert np.array_equal(got, want.astype(t))


def test_one_expert_is_the_dense_product(px_gpu, stream):
    rng = np.random.default_rng(9)
    for M, N, K in ((5, 100, 272), (300, 400, 512)):
        a, w = _normal(px_gpu, rng, M, N, K)
        dense = _run(px_gpu, stream, 16, a, w, M)
        assert np.array_equal(_run(px_gpu, stream, 16, a, w, M, [0, M]), dense)


def test_no_rows(px_gpu, stream):
    px = px_gpu
    a, w = px.F8Rows(0, 0, 0, 64), px.F8Weights(0, 0, 1, 32, 64)
    px.launch_gemm_f8(stream, a, w, px.F16, 0)
    px.launch_gemm_f8_grouped(stream, a, w, 0, 0, 0, px.F16, 0)


@pytest.mark.parametrize("M,N,K", [(3, 600, 4144), (40, 1500, 2064), (300, 512, 1040)])
def test_captured_and_replayed(px_gpu, M, N, K):
    # what lies in device memory changes between the replays: rows, starts, lists
    px = px_gpu
    rng = np.random.default_rng(2)
    s = px.Stream()
    px.bind_workspace(s, 32 << 20)
    a, w = _normal(px, rng, M, N, K, 3)
    dense = px.F8Weights(w.c.ptr, w.s.ptr, 1, N, K)
    dc, de = px.DeviceBuffer(4 * M * N), px.DeviceBuffer(4 * M * N)
    ds, do = px.DeviceBuffer(16), px.DeviceBuffer(4 * M)

    def step():
        px.launch_gemm_f8(s, a.rows, dense, px.F32, dc)
        px.launch_gemm_f8_grouped(s, a.rows, w.weights, ds, do, M, px.F32, de)

    def inputs():
        ds.upload(_groups(rng, 3, M, 1).astype(np.int32))
        do.upload(rng.integers(0, M, M).astype(np.int32))
        a.c.upload(f8.codes_of(rng.uniform(-400, 400, (M, K))))
    inputs()
    step()
    s.synchronize()
    g = Graph(s, step)
    for _ in range(4):
        inputs()
        step()
        s.synchronize()
        want = [b.download(np.float32, (M, N)).copy() for b in (dc, de)]
        for b in (dc, de):
            b.upload(np.full((M, N), 9, np.float32))
        g.replay()
        s.synchronize()
        for b, x in zip((dc, de), want):
            assert np.array_equal(b.download(np.float32, (M, N)), x)
    g.destroy()
    px.bind_workspace(s, 0)
    s.destroy()


def test_rows_past_four_gib(px_gpu, stream):
    # A's and C's offsets pass 32 bits: the last rows of 4.5 GB of codes and of C
    px = px_gpu
    M, N, K = 70000, 20, 65536
    codes, scales = px.DeviceBuffer(M * K), px.DeviceBuffer(M * K // 128 * 4)
    ldc = 40000
    out = px.DeviceBuffer(2 * M * ldc)
    rng = np.random.default_rng(1)
    a, w = _whole(px, rng, 40, N, K)
    codes.zero(stream)
    scales.zero(stream)
    out.zero(stream)
    stream.synchronize()
    from_row = M - 40
    px.check(px.lib().phx_memcpy_d2d(codes.ptr + from_row * K, a.c.ptr, 40 * K))
    px.check(px.lib().phx_memcpy_d2d(scales.ptr + from_row * K // 128 * 4, a.s.ptr, 40 * K // 128 * 4))
    px.launch_gemm_f8(stream, px.F8Rows(codes.ptr, scales.ptr, M, K), w.weights, px.F16, out, 2.0 ** -6,
                      0.0, ldc)
    stream.synchronize()
    got = np.empty((40, ldc), np.float16)
    px.check(px.lib().phx_memcpy_d2h(got.ctypes.data, out.ptr + 2 * from_row * ldc, got.nbytes))
    want = (a.values @ w.values[0].T * 2.0 ** -6).astype(np.float16)
    assert np.array_equal(got[:, :N], want) and (got[:, N:] == 0).all()
