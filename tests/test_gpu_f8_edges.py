"""The operators over 8-bit rows and weights at the ends of what their documentation
allows: offsets past 4 GiB in every operand, the largest strides, the largest lists, both
outputs of the norm over its inputs, a row of zeros without an eps."""
import numpy as np
import pytest

import f8_model as f8
import test_gpu_gemm_f8 as gemm
import test_gpu_f8_rows as rows_of

pytestmark = pytest.mark.gpu


def _put(px, at, array):
    array = np.ascontiguousarray(array)
    px.check(px.lib().phx_memcpy_h2d(at, array.ctypes.data, array.nbytes))


def _get(px, at, t, shape):
    out = np.empty(shape, t)
    px.check(px.lib().phx_memcpy_d2h(out.ctypes.data, at, out.nbytes))
    return out


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("K", [48, 272, 1040, 8208])
def test_norm_h_over_x_and_y_over_r(px_gpu, stream, bits, K):
    px = px_gpu
    dt, t = gemm._t(px, bits)
    rng = np.random.default_rng(K)
    x, r = (rng.standard_normal((9, K)).astype(t) for _ in range(2))
    gain = rng.standard_normal(K).astype(t)
    dx, dr, dg = (px.DeviceBuffer.from_array(v) for v in (x, r, gain))
    codes, scales, rows = rows_of._f8_out(px, 9, K)
    px.launch_norm_f8(stream, dt, dx, dr, dg, dx, dr, rows, 9, K, 1e-5)
    stream.synchronize()
    got = [dx.download(t, (9, K)), dr.download(t, (9, K)), codes.get(), scales.get()]
    rows_of._check_norm(got, x, r, gain, 1e-5)


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("K", [64, 640, 4144])
def test_norm_of_zeros_without_eps(px_gpu, stream, bits, K):
    # f is infinite: codes of 0, no scale and no Y; with an eps everything is 0
    _, t = gemm._t(px_gpu, bits)
    x = np.random.default_rng(1).standard_normal((5, K)).astype(t)
    x[[1, 4]] = 0
    gain = np.ones(K, t)
    h, y, codes, scales = rows_of._norm(px_gpu, stream, bits, x, None, gain, 0.0)
    zero = np.isin(np.arange(5), [1, 4])
    assert np.array_equal(h, x) and (codes[zero] == 0).all()
    assert np.isnan(scales[zero]).all() and np.isnan(y[zero]).all()
    rows_of._check_norm([v[~zero] for v in (h, y, codes, scales)], x[~zero], None, gain, 0.0)
    _, y, codes, scales = rows_of._norm(px_gpu, stream, bits, x, None, gain, 1e-5)
    assert (codes[zero] == 0).all() and (scales[zero] == 0).all() and (y[zero] == 0).all()


@pytest.mark.parametrize("bits", [16, 32])
def test_norm_rows_past_four_gib(px_gpu, stream, bits):
    # X, R, H and Y of three rows 2.4e9 bytes apart
    px = px_gpu
    dt, t = gemm._t(px, bits)
    rng = np.random.default_rng(2)
    M, K, e = 3, 272, bits // 8
    ld = 2_400_000_000 // e
    x, r = (rng.standard_normal((M, K)).astype(t) for _ in range(2))
    gain = rng.standard_normal(K).astype(t)
    bufs = [px.DeviceBuffer(((M - 1) * ld + K) * e) for _ in range(4)]
    for b, v in zip(bufs, (x, r)):
        for m in range(M):
            _put(px, b.ptr + m * ld * e, v[m])
    dg = px.DeviceBuffer.from_array(gain)
    codes, scales, rows = rows_of._f8_out(px, M, K)
    dx, dr, dh, dy = bufs
    px.launch_norm_f8(stream, dt, dx, dr, dg, dh, dy, rows, M, K, 1e-5, ld, ld, ld, ld)
    stream.synchronize()
    h, y = (np.stack([_get(px, b.ptr + m * ld * e, t, K) for m in range(M)]) for b in (dh, dy))
    rows_of._check_norm([h, y, codes.get(), scales.get()], x, r, gain, 1e-5)


@pytest.mark.parametrize("bits", [16, 32])
def test_the_largest_strides(px_gpu, stream, bits):
    # 8-bit rows and their scales 4 MiB apart, 4.6 GB of each: the activation writes them,
    # a product with and one without groups reads them
    px = px_gpu
    dt, t = gemm._t(px, bits)
    rng = np.random.default_rng(3)
    M, K, N, ld = 1100, 144, 40, 1 << 22
    u = rng.standard_normal((M, 2 * K)).astype(t)
    du = px.DeviceBuffer.from_array(u)
    codes, scales = px.DeviceBuffer((M - 1) * ld + K), px.DeviceBuffer(M * ld)
    rows = px.F8Rows(codes.ptr, scales.ptr, M, K, ld, ld // 4)
    px.launch_glu_f8(stream, dt, du, rows)
    stream.synchronize()
    c = np.stack([_get(px, codes.ptr + m * ld, np.uint8, K) for m in range(M)])
    s = np.stack([_get(px, scales.ptr + m * ld, np.float32, 2) for m in range(M)])
    rows_of._check_glu(c, s, rows_of._glu_values(u))
    a = type("A", (), {"rows": rows, "values": f8.row_values(c, s)})
    _, w = gemm._normal(px, rng, 1, N, K, 2)
    starts = np.array([0, 3, M])
    got = gemm._run(px, stream, bits, a, w, M, starts)
    for e in range(2):
        x = a.values[starts[e]:starts[e + 1]]
        want = x @ w.values[e].T
        assert (np.abs(got[starts[e]:starts[e + 1]] - want) <= gemm._bound(want, x, w.values[e], t)).all()
    w.weights = px.F8Weights(w.c.ptr, w.s.ptr, 1, N, K)
    got = gemm._run(px, stream, bits, a, w, M)
    want = a.values @ w.values[0].T
    assert (np.abs(got - want) <= gemm._bound(want, a.values, w.values[0], t)).all()


@pytest.mark.parametrize("bits", [16, 32])
def test_weights_past_four_gib(px_gpu, stream, bits):
    # 19 experts of 256 MiB, of which the last one's rows are whole numbers
    px = px_gpu
    rng = np.random.default_rng(4)
    E, N, K, M = 19, 16400, 16368, 12
    a, _ = gemm._whole(px, rng, M, 1, K, bits=bits)
    codes = px.DeviceBuffer(E * N * K)
    sw = np.ones((E, -(-N // 128), -(-K // 128)), np.float32)
    sw[-1, 5:] = 0.5
    scales = px.DeviceBuffer.from_array(sw)
    codes.zero(stream)
    stream.synchronize()
    last = np.zeros((N, K), np.uint8)
    n = np.r_[0:40, N - 40:N]
    values = np.clip(rng.integers(-2, 3, (n.size, K)), -2, 2)
    last[n] = f8.codes_of(values)
    _put(px, codes.ptr + (E - 1) * N * K, last)
    w = type("W", (), {"weights": px.F8Weights(codes.ptr, scales.ptr, E, N, K)})
    starts = np.full(E + 1, 5)
    starts[0], starts[-1] = 0, M
    got = gemm._run(px, stream, bits, a, w, M, starts)
    assert (got[:5] == 0).all()
    want = np.zeros((M, N))
    want[:, n] = a.values @ (values * np.where(n < 640, 1.0, 0.5)[:, None]).T
    assert np.array_equal(got[5:].astype(np.float64), want[5:])


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("R,K,ld,lds", [((1 << 24) - 1, 128, 128, 4), ((1 << 27) - 1, 16, 16, 4),
                                        (511, 4144, (1 << 22) - 128, 36)])
def test_lists_over_nearly_two_gib(px_gpu, stream, bits, R, K, ld, lds):
    px = px_gpu
    rng = np.random.default_rng(5)
    M, N = 60, 70
    a, w = gemm._whole(px, rng, 8, N, K, 2, bits=bits)
    codes, scales = px.DeviceBuffer((R - 1) * ld + K), px.DeviceBuffer(4 * R * lds)
    kb = -(-K // 128)
    ac = a.c.download(np.uint8, a.c.nbytes)[:8 * K].reshape(8, K)
    sc = a.s.download(np.float32, a.s.nbytes // 4).reshape(8, -1)[:, :kb]
    at = np.array([0, 1, 2, R // 2, R // 2 + 1, R - 3, R - 2, R - 1])
    for i, m in enumerate(at):
        _put(px, codes.ptr + int(m) * ld, ac[i])
        _put(px, scales.ptr + 4 * int(m) * lds, sc[i])
    pick = rng.integers(0, 8, M)
    order = at[pick].astype(np.int64)
    order[[3, 50]] = R, -1
    b = type("A", (), {"rows": px.F8Rows(codes.ptr, scales.ptr, R, K, ld, lds)})
    got = gemm._run(px, stream, bits, b, w, M, [0, 37, M], order)
    x = a.values[pick]
    x[[3, 50]] = 0
    want = np.concatenate([x[:37] @ w.values[0].T, x[37:] @ w.values[1].T])
    assert np.array_equal(got.astype(np.float64), want)
