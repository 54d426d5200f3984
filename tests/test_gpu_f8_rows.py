"""phx_norm_f8 and phx_glu_f8 against 64 bits.  The norm's codes do not depend on
the sum of the squares, so they and the stored rows have to be the exact ones;
scales and Y have the roundings that the header names.  The activation's values are
within 2^-20, so its codes are those of a quotient within 2^-19."""
import numpy as np
import pytest

import f8_model as f8
from hip_graph import Graph

pytestmark = pytest.mark.gpu

GUARD = 64


def _t(px, bits):
    return (px.F16, np.float16) if bits == 16 else (px.F32, np.float32)


class Out:
    """[M, ld] on the device, of which [:, :width] is written, with a guard around."""

    def __init__(self, px, M, width, ld, t, fill):
        self.host = np.full(GUARD + M * ld + GUARD, fill, t)
        self.buf = px.DeviceBuffer.from_array(self.host)
        self.M, self.width, self.ld = M, width, ld
        self.ptr = self.buf.ptr + GUARD * self.host.itemsize

    def get(self):
        got = self.buf.download(self.host.dtype, self.host.shape)
        kept = np.ones(got.shape, bool)
        kept[GUARD:-GUARD].reshape(self.M, self.ld)[:, :self.width] = False
        raw = got.view(np.uint8).reshape(got.size, -1)
        assert np.array_equal(raw[kept], self.host.view(np.uint8).reshape(got.size, -1)[kept]), \
            "stored outside"
        return got[GUARD:-GUARD].reshape(self.M, self.ld)[:, :self.width]


def _pad(x, ld, fill=np.nan):
    out = np.full((x.shape[0], ld), fill, x.dtype)
    out[:, :x.shape[1]] = x
    return out


def _f8_out(px, M, K, pad=0):
    kb = -(-K // 128)
    codes = Out(px, M, K, K + 16 * pad, np.uint8, 0x55)
    scales = Out(px, M, kb, -(-kb // 4) * 4 + 4 * pad, np.float32, 77)
    rows = px.F8Rows(codes.ptr, scales.ptr, M, K, codes.ld if pad else 0, scales.ld if pad else 0)
    return codes, scales, rows


def _norm(px, stream, bits, x, r, gain, eps, want_h=True, want_y=True, want_q=True, pad=0, inplace=None):
    dt, t = _t(px, bits)
    M, K = x.shape
    step = 16 // x.itemsize
    lx, lr = K + pad * step, K + 2 * pad * step
    dx = px.DeviceBuffer.from_array(_pad(x, lx, 7))
    dr = px.DeviceBuffer.from_array(_pad(r, lr, 7)) if r is not None else 0
    dg = px.DeviceBuffer.from_array(gain)
    h = Out(px, M, K, K + 3 * pad * step, t, 77)
    y = Out(px, M, K, K + pad * step, t, 77)
    codes, scales, rows = _f8_out(px, M, K, pad)
    hp, ldh = (h.ptr, h.ld if pad else 0) if want_h else (0, 0)
    if inplace == "x":
        hp, ldh = dx.ptr, lx
    elif inplace == "r":
        hp, ldh = dr.ptr, lr
    px.launch_norm_f8(stream, dt, dx, dr, dg, hp, y.ptr if want_y else 0, rows if want_q else None,
                      M, K, eps, lx if pad else 0, lr if pad and r is not None else 0, ldh,
                      y.ld if pad and want_y else 0)
    stream.synchronize()
    if inplace:
        ld = lx if inplace == "x" else lr
        got_h = (dx if inplace == "x" else dr).download(t, (M, ld))
        assert (got_h[:, K:] == 7).all()
        got_h = got_h[:, :K]
    else:
        got_h = h.get()
        if not want_h:
            assert (got_h == 77).all()
    got = [got_h, y.get(), codes.get(), scales.get()]
    if not want_y:
        assert (got[1] == 77).all()
    if not want_q:
        assert (got[2] == 0x55).all() and (got[3] == 77).all()
    return got


def _check_norm(got, x, r, gain, eps, want_h=True, want_y=True, want_q=True):
    t = x.dtype
    h, prod, factor = f8.norm(x, r, gain, eps)
    q, a = f8.quotients(prod)
    if want_h:
        assert np.array_equal(got[0], h)
    if want_q:
        assert np.array_equal(got[2], f8.codes_of(q))
        want = a * factor / 448
        # one rounding to f32 of a quotient in 64 bits, and the sum's order
        assert (np.abs(got[3] - want) <= np.abs(want) * (2.0 ** -24 + 2.0 ** -40) + 2.0 ** -150).all()
    if want_y:
        want = prod.astype(np.float64) * factor
        # the factor and the product in f32, then the type
        off = np.abs(want) * 2.0 ** -23 * (1 + 2.0 ** -20)
        half = np.finfo(t).eps / 2 if t == np.float16 else 0
        tiny = 2.0 ** -25 if t == np.float16 else 2.0 ** -149
        assert (np.abs(got[1] - want) <= (np.abs(want) + off) * half + off + tiny).all()


# lengths at the edges of every form: one 16-byte chunk a thread up to eight
LENGTHS = [16, 112, 128, 144, 512, 528, 1040, 2048, 2064, 4096, 4144, 8192, 8208, 16384, 16400, 32768]


@pytest.mark.parametrize("K", LENGTHS)
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("M", [1, 6])
def test_norm(px_gpu, stream, bits, K, M):
    rng = np.random.default_rng(K + M + bits)
    _, t = _t(px_gpu, bits)
    x = (rng.standard_normal((M, K)) * 10.0 ** rng.uniform(-2, 2, (M, 1))).astype(t)
    r = rng.standard_normal((M, K)).astype(t)
    gain = (1 + 0.2 * rng.standard_normal(K)).astype(t)
    for res in (r, None):
        got = _norm(px_gpu, stream, bits, x, res, gain, 1e-5)
        _check_norm(got, x, res, gain, 1e-5)


@pytest.mark.parametrize("K", [16, 32, 48, 64, 80, 112, 128, 144, 256, 272])
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("M", [3, 127, 300])
def test_norm_short_rows(px_gpu, stream, bits, K, M):
    # several rows a wave, the last ones' lanes idle
    rng = np.random.default_rng(K * M + bits)
    _, t = _t(px_gpu, bits)
    x = (rng.standard_normal((M, K)) * 10.0 ** rng.uniform(-2, 2, (M, 1))).astype(t)
    r = rng.standard_normal((M, K)).astype(t)
    gain = (1 + 0.2 * rng.standard_normal(K)).astype(t)
    _check_norm(_norm(px_gpu, stream, bits, x, r, gain, 1e-5, pad=1), x, r, gain, 1e-5)


def test_norm_short_rows_of_every_size(px_gpu, stream):
    # neighbours in a wave, of which some have a factor that no f32 holds
    rng = np.random.default_rng(31)
    exponents = np.array([0, -146, 3, 124, -130, 0, 20])[np.arange(60) % 7]
    x = np.ldexp(rng.standard_normal((60, 64)), exponents[:, None]).astype(np.float32)
    gain = np.ones(64, np.float32)
    got = _norm(px_gpu, stream, 32, x, None, gain, 0.0)
    _check_norm(got, x, None, gain, 0.0)
    for m in (0, 5, 6):  # a row's bits are its own
        alone = _norm(px_gpu, stream, 32, x[m:m + 1], None, gain, 0.0)
        for a, b in zip(alone, got):
            assert np.array_equal(a[0], b[m])


@pytest.mark.parametrize("bits", [16, 32])
def test_norm_strides_and_outputs(px_gpu, stream, bits):
    rng = np.random.default_rng(2)
    _, t = _t(px_gpu, bits)
    for M, K in ((5, 272), (3, 2576), (2, 9008)):
        x, r = (rng.standard_normal((M, K)).astype(t) for _ in range(2))
        gain = rng.standard_normal(K).astype(t)
        for kw in (dict(), dict(want_h=False), dict(want_y=False), dict(want_q=False),
                   dict(want_h=False, want_y=False), dict(want_h=False, want_q=False)):
            got = _norm(px_gpu, stream, bits, x, r, gain, 1e-6, pad=1, **kw)
            _check_norm(got, x, r, gain, 1e-6, **kw)
        for where in ("x", "r"):
            got = _norm(px_gpu, stream, bits, x, r, gain, 1e-6, pad=1, inplace=where)
            _check_norm(got, x, r, gain, 1e-6)


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("K", [528, 2064, 20000])
def test_norm_with_y_in_place(px_gpu, stream, bits, K):
    # Y over X, and H over R
    px = px_gpu
    dt, t = _t(px, bits)
    rng = np.random.default_rng(K)
    x, r = (rng.standard_normal((5, K)).astype(t) for _ in range(2))
    gain = rng.standard_normal(K).astype(t)
    dx, dr, dg = (px.DeviceBuffer.from_array(v) for v in (x, r, gain))
    codes, scales, rows = _f8_out(px, 5, K)
    px.launch_norm_f8(stream, dt, dx, dr, dg, dr, dx, rows, 5, K, 1e-5)
    stream.synchronize()
    got = [dr.download(t, (5, K)), dx.download(t, (5, K)), codes.get(), scales.get()]
    _check_norm(got, x, r, gain, 1e-5)


@pytest.mark.parametrize("bits", [16, 32])
def test_norm_codes_at_ties(px_gpu, stream, bits):
    # 448 in every block, so that a value is its own quotient: all codes' values,
    # the middles between them, and what is next to those
    _, t = _t(px_gpu, bits)
    v = f8.VALUES[:127]
    mid = (v[1:] + v[:-1]) / 2
    q = np.concatenate([v, mid, *(np.nextafter(mid.astype(t), t(s)).astype(np.float64)
                                  for s in (0, 1000))])
    q = np.concatenate([q, -q])
    q = np.concatenate([q, np.zeros(-q.size % 127)]).reshape(-1, 127)
    x = np.concatenate([q, np.full((q.shape[0], 1), 448.0)], 1).reshape(1, -1).astype(t)
    gain = np.ones(x.shape[1], t)
    got = _norm(px_gpu, stream, bits, x, None, gain, 1e-5)
    _check_norm(got, x, None, gain, 1e-5)
    # quotients of small whole numbers: many ties that are no values of t
    rng = np.random.default_rng(1)
    x = rng.integers(-40, 41, (64, 2048)).astype(t)
    for scale in (1.0, 3.0, 0.21875):
        gain = np.full(2048, scale, t)
        _check_norm(_norm(px_gpu, stream, bits, x, None, gain, 1e-5), x, None, gain, 1e-5)


@pytest.mark.parametrize("exponent", [-146, -130, -126, -110, -101, -99, 60, 99, 101, 110])
def test_norm_tiny_and_large_f32(px_gpu, stream, exponent):
    rng = np.random.default_rng(200 + exponent)
    x = np.ldexp(rng.standard_normal((3, 640)), exponent).astype(np.float32)
    gain = (1 + 0.2 * rng.standard_normal(640)).astype(np.float32)
    got = _norm(px_gpu, stream, 32, x, None, gain, 0.0, want_y=abs(exponent) < 105)
    _check_norm(got, x, None, gain, 0.0, want_y=abs(exponent) < 105)


@pytest.mark.parametrize("exponent", [-146, -135, -128, -126, 110, 124])
def test_norm_y_where_no_f32_holds_the_factor(px_gpu, stream, exponent):
    rng = np.random.default_rng(300 + exponent)
    x = np.ldexp(rng.standard_normal((3, 640)), exponent).astype(np.float32)
    gain = np.ones(640, np.float32)
    _check_norm(_norm(px_gpu, stream, 32, x, None, gain, 0.0), x, None, gain, 0.0)


@pytest.mark.parametrize("bits", [16, 32])
def test_norm_zeros_infinities_and_nan(px_gpu, stream, bits):
    px = px_gpu
    _, t = _t(px, bits)
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 400)).astype(t)
    gain = np.ones(400, t)
    clean = _norm(px, stream, bits, x, None, gain, 1e-5)
    x[1] = 0
    x[2, 128:256] = 0
    x[3, 130], x[4, 399] = np.nan, np.inf
    got = _norm(px, stream, bits, x, None, gain, 1e-5)
    for a, b in zip(got, clean):
        assert np.array_equal(a[[0, 5]], b[[0, 5]])
    assert (got[1][1] == 0).all() and (got[2][1] == 0).all() and (got[3][1] == 0).all()
    assert (got[2][2, 128:256] == 0).all() and got[3][2, 1] == 0 and (got[3][2, [0, 2, 3]] > 0).all()
    nan = np.isnan(f8.VALUES[got[2]])
    assert nan[3, 128:256].all() and nan[4, 384:].all()
    assert np.isnan(got[1][3]).all() and np.isnan(got[3][3]).all()
    assert np.isnan(got[3][4, 3]) and np.isnan(got[1][4, 399])
    # what an infinity leaves of its row is the formula's zeros
    assert (got[1][4, :399] == 0).all() and (got[3][4, :3] == 0).all()


def test_norm_sum_of_large_f32_squares(px_gpu, stream):
    # squares beyond f32: summed in 64 bits
    x = np.full((2, 256), 1e25, np.float32)
    x[:, ::2] = -3e25
    gain = np.ones(256, np.float32)
    _check_norm(_norm(px_gpu, stream, 32, x, None, gain, 1e-5), x, None, gain, 1e-5)


def test_norm_many_rows(px_gpu, stream):
    rng = np.random.default_rng(9)
    x, r = (rng.standard_normal((2051, 528)).astype(np.float16) for _ in range(2))
    gain = rng.standard_normal(528).astype(np.float16)
    _check_norm(_norm(px_gpu, stream, 16, x, r, gain, 1e-5), x, r, gain, 1e-5)


def test_no_rows(px_gpu, stream):
    px = px_gpu
    px.launch_norm_f8(stream, px.F16, 0, 0, 0, 0, 0, px.F8Rows(0, 0, 0, 64), 0, 64, 1e-5)
    px.launch_glu_f8(stream, px.F16, 0, px.F8Rows(0, 0, 0, 64))


# ---------------------------------------------------------------- the gated activation
def _glu(px, stream, bits, u, pad=0):
    dt, _ = _t(px, bits)
    M, K = u.shape[0], u.shape[1] // 2
    ldu = 2 * K + pad * (16 // u.itemsize)
    du = px.DeviceBuffer.from_array(_pad(u, ldu))
    codes, scales, rows = _f8_out(px, M, K, pad)
    px.launch_glu_f8(stream, dt, du, rows, ldu if pad else 0)
    stream.synchronize()
    return codes.get(), scales.get()


def _glu_values(u):
    u = u.astype(np.float64)
    gate, value = np.split(u, 2, 1)
    with np.errstate(over="ignore", invalid="ignore"):
        return gate / (1 + np.exp(-gate)) * value


def _check_glu(codes, scales, v):
    q, a = f8.quotients(v)
    lo, hi = f8.codes_of(np.clip(q * (1 - 2.0 ** -19), -448, 448)), \
        f8.codes_of(np.clip(q * (1 + 2.0 ** -19), -448, 448))
    assert ((codes == lo) | (codes == hi)).all()
    # (codes that differ stand next to a tie: few values do)
    assert (lo != hi).mean() < 2.0 ** -10 or v.size < 4096
    want = a / 448
    assert (np.abs(scales - want) <= want * (2.0 ** -20 + 2.0 ** -23) + 2.0 ** -149).all()


@pytest.mark.parametrize("M,K", [(1, 16), (3, 112), (7, 128), (5, 144), (2, 4096), (33, 5520), (300, 1040)])
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("pad", [0, 1])
def test_glu(px_gpu, stream, bits, M, K, pad):
    rng = np.random.default_rng(M + K)
    _, t = _t(px_gpu, bits)
    u = (rng.standard_normal((M, 2 * K)) * 10.0 ** rng.uniform(-2, 1, (M, 1))).astype(t)
    _check_glu(*_glu(px_gpu, stream, bits, u, pad), _glu_values(u))


@pytest.mark.parametrize("bits", [16, 32])
def test_glu_gates_of_every_size(px_gpu, stream, bits):
    # one gate a block, as the others would hide the small ones' codes
    _, t = _t(px_gpu, bits)
    most = 60000.0 if bits == 16 else 3e38
    g = np.concatenate([np.linspace(-80, 80, 161), [most, 0.0, 1e-3, -1e-3, -1e-7, 200.0, 1e4, 88.0, 89.0]])
    u = np.zeros((g.size, 256), t)
    u[:, 3], u[:, 128 + 3] = g, 1.0
    u[g == most, 131] = 0.5
    codes, scales = _glu(px_gpu, stream, bits, u)
    _check_glu(codes, scales, _glu_values(u))


@pytest.mark.parametrize("bits", [16, 32])
def test_glu_infinities_and_nan(px_gpu, stream, bits):
    rng = np.random.default_rng(3)
    _, t = _t(px_gpu, bits)
    u = rng.standard_normal((5, 2 * 272)).astype(t)
    clean = _glu(px_gpu, stream, bits, u)
    u[0, 5], u[1, 272 + 130], u[2, 260], u[3, 272 + 3] = np.nan, np.nan, np.inf, -np.inf
    codes, scales = _glu(px_gpu, stream, bits, u)
    bad = np.zeros((5, 3), bool)
    bad[[0, 1, 2, 3], [0, 1, 2, 0]] = True
    assert np.array_equal(np.isnan(scales), bad)
    each = np.repeat(bad, 128, 1)[:, :272]
    assert np.array_equal(np.isnan(f8.VALUES[codes]), each)
    assert np.array_equal(codes[~each], clean[0][~each]) and np.array_equal(scales[~bad], clean[1][~bad])


def test_captured_and_replayed(px_gpu):
    px = px_gpu
    rng = np.random.default_rng(6)
    s, M, K = px.Stream(), 40, 1040
    dx, dr, dg, dh = (px.DeviceBuffer(2 * M * K) for _ in range(4))
    codes, scales, rows = _f8_out(px, M, K)
    half, hs, hrows = _f8_out(px, M, K // 2 // 16 * 16)
    gain = rng.standard_normal(K).astype(np.float16)
    dg.upload(gain)

    def step():
        px.launch_norm_f8(s, px.F16, dx, dr, dg, dh, 0, rows, M, K, 1e-5)
        px.launch_glu_f8(s, px.F16, dh, hrows, K)
    step()
    s.synchronize()
    g = Graph(s, step)
    for _ in range(4):
        x, r = (rng.standard_normal((M, K)).astype(np.float16) for _ in range(2))
        dx.upload(x)
        dr.upload(r)
        g.replay()
        s.synchronize()
        got = [dh.download(np.float16, (M, K)), None, codes.get(), scales.get()]
        _check_norm(got, x, r, gain, 1e-5, want_y=False)
        again = [half.get().copy(), hs.get().copy()]
        step()
        s.synchronize()
        assert np.array_equal(half.get(), again[0]) and np.array_equal(hs.get(), again[1])
    g.destroy()
    s.destroy()
