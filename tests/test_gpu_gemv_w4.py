"""phx_gemv_w4 against 64 bits.  With small whole numbers and scales that are
powers of two every product and partial sum is exact, so the result has to be
the exact one: any wrong index, nibble, group or mask shows.  With normal
inputs the bound is the arithmetic's: f32 sums of K products, one rounding of
the output."""
import numpy as np
import pytest

from hip_graph import Graph

pytestmark = pytest.mark.gpu

GUARD = 64  # elements around every output


def _pack(px, stream, codes):
    K, N = codes.shape
    packed = px.DeviceBuffer(px.w4_packed_bytes(N, K))
    dc = px.DeviceBuffer.from_array(codes)
    px.w4_pack(stream, dc, packed, N, K)
    stream.synchronize()
    return packed


def _np(px, dtype):
    return np.float16 if dtype == px.F16 else np.float32


def _run(px, stream, dtype, a, codes, scales, zeros, group, alpha=1.0, beta=0.0, c=None, lda=0,
         ldc=0):
    """The C rows; what lies between and around them has to stay."""
    t = _np(px, dtype)
    (M, K), N = a.shape, codes.shape[1]
    lda, ldc = lda or K, ldc or N
    host = np.full((M, lda), np.nan, t)
    host[:, :K] = a
    out = np.full(GUARD + M * ldc + GUARD, 77, t)
    view = out[GUARD:GUARD + M * ldc].reshape(M, ldc)
    if c is not None:
        view[:, :N] = c
    elif beta == 0.0:
        view[:, :N] = np.nan  # not read
    bufs = [px.DeviceBuffer.from_array(x) for x in (host, scales.astype(np.float16), out)]
    dz = px.DeviceBuffer.from_array(zeros) if zeros is not None else None
    w = _pack(px, stream, codes)
    px.launch_gemv_w4(stream, dtype, bufs[0], w, bufs[1], dz or 0, bufs[2].ptr + GUARD * out.itemsize,
                      M, N, K, group, alpha, beta, lda, ldc)
    stream.synchronize()
    got = bufs[2].download(t, out.shape)
    kept = np.ones(out.shape, bool)
    kept[GUARD:GUARD + M * ldc].reshape(M, ldc)[:, :N] = False
    assert np.array_equal(got[kept], out[kept]), "stored outside C"
    return got[GUARD:GUARD + M * ldc].reshape(M, ldc)[:, :N]


def _weights(codes, scales, zeros, group):
    g = np.arange(codes.shape[0]) // group
    z = 8 if zeros is None else zeros.astype(np.int64)[g]
    return (codes.astype(np.int64) - z) * scales.astype(np.float64)[g]


SHAPES = [(1, 1, 8), (1, 16, 128), (2, 17, 136), (3, 5, 24), (15, 33, 120), (16, 16, 256),
          (17, 40, 392), (33, 100, 72), (64, 15, 520), (48, 257, 1032), (1, 1000, 4136), (4, 64, 8192),
          (64, 130, 2056), (5, 4099, 64), (1, 31, 16384)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_whole_numbers_are_exact(px_gpu, stream, bits, M, N, K, group):
    px = px_gpu
    rng = np.random.default_rng(M * 7 + N * 3 + K + group)
    groups = -(-K // group)
    dtype = px.F16 if bits == 16 else px.F32
    codes = rng.integers(0, 16, (K, N)).astype(np.uint8)
    zeros = rng.integers(0, 16, (groups, N)).astype(np.uint8) if M % 2 else None
    scales = 2.0 ** rng.integers(-2, 2, (groups, N))
    # f16: few non-zero elements, so that the sums stay whole and below 2048
    # quarters; f32: whole numbers of up to 10 bits with sums below 2^24
    # quarters
    a = np.zeros((M, K))
    for m in range(M):
        at = rng.choice(K, min(K, 6 if bits == 16 else 200), replace=False)
        a[m, at] = rng.integers(-2, 3, at.size) if bits == 16 else rng.integers(-600, 601, at.size)
    want = a @ _weights(codes, scales, zeros, group)
    got = _run(px, stream, dtype, a, codes, scales, zeros, group)
    assert np.array_equal(got.astype(np.float64), want)


def _bound(want, mag, K, t, alpha=1.0, extra=0.0):
    """Half a step of the output, and f32's of K products, their scales and
    sums, alpha and beta."""
    half = np.finfo(t).eps / 2
    inner = ((K + 8) * mag * abs(alpha) + 2 * extra + np.abs(want)) * 2.0 ** -24
    tiny = 2.0 ** -25 if t == np.float16 else 2.0 ** -149
    return (np.abs(want) + inner) * half + inner + tiny


@pytest.mark.parametrize("M,N,K", [(1, 48, 4096), (5, 1000, 4136), (16, 333, 520), (64, 100, 2048),
                                   (23, 18, 8192)])
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("group", [32, 128])
def test_normal_inputs(px_gpu, stream, bits, M, N, K, group):
    px = px_gpu
    rng = np.random.default_rng(K + N)
    groups = -(-K // group)
    dtype = px.F16 if bits == 16 else px.F32
    t = _np(px, dtype)
    codes = rng.integers(0, 16, (K, N)).astype(np.uint8)
    zeros = rng.integers(0, 256, (groups, N)).astype(np.uint8)
    scales = (rng.random((groups, N)) * 0.01 + 1e-4).astype(np.float16)
    # rows of very different magnitudes
    a = (rng.standard_normal((M, K)) * 10.0 ** rng.uniform(-2, 1, (M, 1))).astype(t)
    w = _weights(codes, scales, zeros, group)
    want, mag = a.astype(np.float64) @ w, np.abs(a.astype(np.float64)) @ np.abs(w)
    got = _run(px, stream, dtype, a, codes, scales, zeros, group, lda=K + 24, ldc=N + 3)
    assert (np.abs(got - want) <= _bound(want, mag, K, t)).all()


def test_f32_operands_keep_all_their_bits(px_gpu, stream):
    # one non-zero element of 24 bits per row against weights of 1: the output
    # is that element, whatever its exponent
    px = px_gpu
    rng = np.random.default_rng(11)
    M, N, K = 64, 20, 264
    a = np.zeros((M, K), np.float32)
    val = (rng.integers(1 << 23, 1 << 24, M) * 2.0 ** rng.integers(-120, 100, M)).astype(np.float32)
    a[np.arange(M), rng.integers(0, K, M)] = val * np.where(rng.random(M) < 0.5, -1, 1)
    codes = np.full((K, N), 9, np.uint8)
    got = _run(px, stream, px.F32, a, codes, np.ones((9, N)), None, 32)
    assert np.array_equal(got, np.repeat(a.sum(1, keepdims=True), N, 1))


@pytest.mark.parametrize("bits", [16, 32])
def test_alpha_and_beta(px_gpu, stream, bits):
    px = px_gpu
    rng = np.random.default_rng(3)
    M, N, K = 6, 50, 640
    dtype = px.F16 if bits == 16 else px.F32
    t = _np(px, dtype)
    codes = rng.integers(0, 16, (K, N)).astype(np.uint8)
    scales = (rng.random((10, N)) * 0.1).astype(np.float16)
    a, c = rng.standard_normal((M, K)).astype(t), rng.standard_normal((M, N)).astype(t)
    w = _weights(codes, scales, None, 64)
    want = 0.5 * (a.astype(np.float64) @ w) - 1.5 * c.astype(np.float64)
    mag = np.abs(a.astype(np.float64)) @ np.abs(w)
    got = _run(px, stream, dtype, a, codes, scales, None, 64, 0.5, -1.5, c)
    assert (np.abs(got - want) <= _bound(want, mag, K, t, 0.5, 1.5 * np.abs(c))).all()
    # alpha 0 and a C of NaN: not read with beta 0
    assert (_run(px, stream, dtype, a, codes, scales, None, 64, 0.0, 0.0) == 0).all()


@pytest.mark.parametrize("bits", [16, 32])
def test_a_row_of_infinities_stays_in_its_row(px_gpu, stream, bits):
    px = px_gpu
    rng = np.random.default_rng(5)
    M, N, K = 7, 40, 264
    dtype = px.F16 if bits == 16 else px.F32
    codes = rng.integers(9, 16, (K, N)).astype(np.uint8)  # weights above 0
    scales = np.full((9, N), 0.25)
    a = rng.integers(-2, 3, (M, K)).astype(_np(px, dtype))
    clean = _run(px, stream, dtype, a, codes, scales, None, 32)
    a[2, 9], a[4, 200] = np.nan, np.inf
    got = _run(px, stream, dtype, a, codes, scales, None, 32)
    keep = [0, 1, 3, 5, 6]
    assert np.array_equal(got[keep], clean[keep])
    assert np.isnan(got[2]).all() and not np.isfinite(got[4]).any()


def test_no_rows(px_gpu, stream):
    px_gpu.launch_gemv_w4(stream, px_gpu.F16, 0, 0, 0, 0, 0, 0, 16, 128, 32)


def test_quantised_weights_stand_for_the_weights(px_gpu, stream):
    px = px_gpu
    rng = np.random.default_rng(8)
    b = rng.standard_normal((200, 30)) / 14
    codes, scales, zeros = px.w4_quantize(b, 32)
    a = rng.standard_normal((3, 200)).astype(np.float16)
    got = _run(px, stream, px.F16, a, codes, scales, zeros, 32)
    w = _weights(codes, scales, zeros, 32)
    a = a.astype(np.float64)
    assert (np.abs(got - a @ w) <= _bound(a @ w, np.abs(a) @ np.abs(w), 200, np.float16)).all()
    assert np.abs(w - b).max() <= scales.astype(np.float64).max() * (1 + 15 * 2.0 ** -11)


# M at the edges of the row tiles; K that splits in 2 and in 4 chunks, the last
# of them short
SPLIT = [(17, 1000, 4136), (32, 33, 2056), (33, 1000, 4136), (48, 65, 1160), (64, 2500, 2048),
         (64, 16, 16384), (24, 130, 9000), (33, 1500, 8192), (64, 1290, 4400), (47, 2600, 16384)]


@pytest.mark.parametrize("M,N,K", SPLIT)
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("parts", [0, 1.9, 2, 3.9, 4, 9])
def test_split_over_k(px_gpu, bits, M, N, K, parts):
    # a workspace of so many parts: what lies behind it has to stay
    px = px_gpu
    rng = np.random.default_rng(M + N + K)
    dtype = px.F16 if bits == 16 else px.F32
    t = _np(px, dtype)
    codes = rng.integers(0, 16, (K, N)).astype(np.uint8)
    scales = (rng.random((-(-K // 64), N)) * 0.01).astype(np.float16)
    a, c = rng.standard_normal((M, K)).astype(t), rng.standard_normal((M, N)).astype(t)
    w = _weights(codes, scales, None, 64)
    want = 0.5 * (a.astype(np.float64) @ w) + c
    mag = np.abs(a.astype(np.float64)) @ np.abs(w)
    room = int(parts * M * N) * 4
    ws = px.DeviceBuffer.from_array(np.full(room + 4096, 0xAB, np.uint8))
    s = px.Stream()
    if room:
        px.set_workspace(s, ws.ptr, room)
    got = _run(px, s, dtype, a, codes, scales, None, 64, 0.5, 1.0, c)
    px.set_workspace(s, 0, 0)
    s.destroy()
    assert (np.abs(got - want) <= _bound(want, mag, K, t, 0.5, np.abs(c))).all()
    assert (ws.download(np.uint8, room + 4096)[room:] == 0xAB).all()


@pytest.mark.parametrize("M,N,K", [(40, 600, 4136), (40, 1500, 8192)])
def test_captured_and_replayed(px_gpu, M, N, K):
    px = px_gpu
    rng = np.random.default_rng(2)
    codes = rng.integers(0, 16, (K, N)).astype(np.uint8)
    scales = (rng.random((-(-K // 32), N)) * 0.01).astype(np.float16)
    s = px.Stream()
    px.bind_workspace(s, 16 * M * N)
    w, ds = _pack(px, s, codes), px.DeviceBuffer.from_array(scales)
    da, dc = px.DeviceBuffer(2 * M * K), px.DeviceBuffer(2 * M * N)

    def step(m):
        px.launch_gemv_w4(s, px.F16, da, w, ds, 0, dc, m, N, K, 32)
    step(M)
    s.synchronize()
    graphs = [Graph(s, lambda: step(M)), Graph(s, lambda: step(20))]
    for _ in range(4):
        da.upload(rng.standard_normal((M, K)).astype(np.float16))
        for g, m in zip(graphs, (M, 20)):
            step(m)
            s.synchronize()
            want = dc.download(np.float16, (m, N)).copy()
            dc.upload(np.full((M, N), 9, np.float16))
            g.replay()
            s.synchronize()
            assert np.array_equal(dc.download(np.float16, (M, N))[:m], want)
    for g in graphs:
        g.destroy()
    px.bind_workspace(s, 0)
    s.destroy()


@pytest.mark.parametrize("M,N,K", [(1, 8190, 392), (16, 5000, 264), (7, 20001, 136), (16, 4111, 2056),
                                   (3, 16400, 8)])
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_many_columns(px_gpu, stream, bits, M, N, K, group):
    # the tiles of 32 and 64 columns, the last of them short
    px = px_gpu
    rng = np.random.default_rng(N)
    dtype = px.F16 if bits == 16 else px.F32
    t = _np(px, dtype)
    codes = rng.integers(0, 16, (K, N)).astype(np.uint8)
    scales = (rng.random((-(-K // group), N)) * 0.01).astype(np.float16)
    zeros = rng.integers(0, 16, scales.shape).astype(np.uint8)
    a = rng.standard_normal((M, K)).astype(t)
    w = _weights(codes, scales, zeros, group)
    want, mag = a.astype(np.float64) @ w, np.abs(a.astype(np.float64)) @ np.abs(w)
    got = _run(px, stream, dtype, a, codes, scales, zeros, group)
    assert (np.abs(got - want) <= _bound(want, mag, K, t)).all()


@pytest.mark.parametrize("M,N,K", [(3, 40, 520), (40, 300, 1032)])
@pytest.mark.parametrize("bits,exponent", [(16, -8), (16, -14), (16, -17), (16, -20), (32, 40), (32, -104),
                                           (32, -112), (32, -120), (32, -126), (32, -135)])
def test_rows_of_tiny_and_large_elements(px_gpu, stream, bits, exponent, M, N, K):
    # what an f32 element has below 2^-126 counts as 0; f16 elements enter whole,
    # subnormal ones too
    px = px_gpu
    rng = np.random.default_rng(M + 200 - exponent)
    dtype = px.F16 if bits == 16 else px.F32
    t = _np(px, dtype)
    codes = rng.integers(0, 16, (K, N)).astype(np.uint8)
    scales = np.full((-(-K // 32), N), 64.0)
    a = np.ldexp(rng.standard_normal((M, K)), exponent).astype(t)
    w = _weights(codes, scales, None, 32)
    want, mag = a.astype(np.float64) @ w, np.abs(a.astype(np.float64)) @ np.abs(w)
    got = _run(px, stream, dtype, a, codes, scales, None, 32)
    lost = np.abs(w).sum(0) * 2.0 ** -126 if bits == 32 else 0.0
    # (of a sum of f16 subnormals the matrix instructions keep 20 bits: one
    # rounding in every 32 products)
    lost = lost + (mag * 2.0 ** -20 if bits == 16 else 0.0)
    assert (np.abs(got - want) <= _bound(want, mag, K, t) + lost).all()
