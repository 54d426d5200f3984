"""What the operators over 8-bit rows and weights refuse, before any device is
touched: without one a good call ends in PHX_E_NOT_INIT and a bad one in
PHX_E_INVALID.  And the host's quantiser of weights."""
import numpy as np
import pytest

import f8_model as f8
import phobos_amd as px

A = 1 << 20  # an address that passes the checks; nothing is launched
BIG = 1 << 50


@pytest.fixture(autouse=True, scope="module")
def _no_device():
    if px._INIT:
        pytest.skip("the library is initialised on a device in this process")


def _rc(f):
    try:
        f()
    except px.PhxError as e:
        return e.code
    return 0


def _rows(**kw):
    d = dict(codes=A, scales=A, rows=3, k=144, ld=0, lds=0)
    d.update(kw)
    return px.F8Rows(*d.values())


def _weights(**kw):
    d = dict(codes=A, scales=A, experts=1, n=5, k=144)
    d.update(kw)
    return px.F8Weights(*d.values())


BAD_ROWS = [dict(codes=0), dict(scales=0), dict(codes=A + 8), dict(scales=A + 4), dict(rows=-1),
            dict(rows=1 << 31), dict(ld=128), dict(ld=152), dict(ld=-144), dict(ld=BIG), dict(lds=1),
            dict(lds=3), dict(lds=6), dict(lds=-4), dict(lds=BIG),
            dict(lds=(1 << 20) + 4)]


def _norm(rows=None, **kw):
    a = dict(dtype=px.F16, x=A, r=A, gain=A, h=A, y=A, M=3, K=144, eps=1e-5, ldx=0, ldr=0, ldh=0, ldy=0)
    a.update(kw)
    q = _rows(**{"rows": a["M"], "k": a["K"], **(rows or {})}) if rows != "none" else None
    return _rc(lambda: px.launch_norm_f8(None, a["dtype"], a["x"], a["r"], a["gain"], a["h"], a["y"], q,
                                         a["M"], a["K"], a["eps"], a["ldx"], a["ldr"], a["ldh"],
                                         a["ldy"]))


@pytest.mark.parametrize("ok", [
    {}, {"r": 0}, {"h": 0}, {"y": 0}, {"rows": "none"}, {"r": 0, "h": 0, "y": 0}, {"dtype": px.F32},
    {"K": 16}, {"K": 32768}, {"M": 0, "x": 0, "gain": 0, "r": 0, "h": 0, "y": 0}, {"eps": 0.0},
    {"M": 0, "rows": {"codes": 0, "scales": 0}}, {"ldx": 152, "ldr": 160, "ldh": 168, "ldy": 176},
    {"dtype": px.F32, "ldx": 148}, {"rows": {"ld": 160, "lds": 8}}, {"M": 4_000_000}])
def test_norm_takes(ok):
    assert _norm(**ok) == px.PHX_E_NOT_INIT


@pytest.mark.parametrize("bad", [
    {"dtype": 2}, {"dtype": -1}, {"M": -1}, {"M": 1 << 31}, {"M": (1 << 31) - 1, "K": 4096}, {"K": 0}, {"K": 8},
    {"K": 136}, {"K": -16}, {"K": 32784}, {"K": BIG}, {"eps": -1e-5}, {"eps": float("nan")},
    {"eps": float("inf")}, {"x": 0}, {"gain": 0}, {"x": A + 8}, {"r": A + 2}, {"gain": A + 8},
    {"h": A + 4}, {"y": A + 8}, {"ldx": 136}, {"ldx": 148}, {"ldr": 100}, {"ldh": -144}, {"ldy": BIG},
    {"dtype": px.F32, "ldx": 146}, {"rows": "none", "y": 0}, {"rows": {"rows": 4}}, {"rows": {"k": 160}},
    *({"rows": x} for x in BAD_ROWS)])
def test_norm_refuses(bad):
    assert _norm(**bad) == px.PHX_E_INVALID
    assert "norm_f8" in px.lib().phx_last_error().decode()


def _glu(rows=None, **kw):
    a = dict(dtype=px.F16, u=A, ldu=0)
    a.update(kw)
    q = _rows(**(rows or {})) if rows != "none" else None
    return _rc(lambda: px.launch_glu_f8(None, a["dtype"], a["u"], q, a["ldu"]))


@pytest.mark.parametrize("ok", [{}, {"dtype": px.F32}, {"ldu": 296}, {"dtype": px.F32, "ldu": 292},
                                {"rows": {"k": 1 << 22, "rows": 1}},
                                {"rows": {"rows": 0, "codes": 0, "scales": 0}, "u": 0}])
def test_glu_takes(ok):
    assert _glu(**ok) == px.PHX_E_NOT_INIT


@pytest.mark.parametrize("bad", [
    {"dtype": 2}, {"u": 0}, {"u": A + 8}, {"ldu": 280}, {"ldu": 292}, {"ldu": -288}, {"ldu": BIG},
    {"rows": "none"}, {"rows": {"k": 0}}, {"rows": {"k": 8}}, {"rows": {"k": 136}}, {"rows": {"k": -16}},
    {"rows": {"k": (1 << 22) + 16}}, {"rows": {"rows": (1 << 31) - 1, "k": 1 << 20}},
    *({"rows": x} for x in BAD_ROWS)])
def test_glu_refuses(bad):
    assert _glu(**bad) == px.PHX_E_INVALID
    assert "glu_f8" in px.lib().phx_last_error().decode()


def _gemm(rows=None, weights=None, **kw):
    a = dict(dtype=px.F16, c=A, alpha=1.0, beta=0.0, ldc=0)
    a.update(kw)
    r = _rows(**(rows or {})) if rows != "none" else None
    w = _weights(**(weights or {})) if weights != "none" else None
    return _rc(lambda: px.launch_gemm_f8(None, r, w, *a.values()))


def _grouped(rows=None, weights=None, **kw):
    a = dict(starts=A, order=A, M=7, dtype=px.F16, c=A, alpha=1.0, beta=0.0, ldc=0)
    a.update(kw)
    r = _rows(**(rows or {})) if rows != "none" else None
    w = _weights(**{"experts": 4, **(weights or {})}) if weights != "none" else None
    return _rc(lambda: px.launch_gemm_f8_grouped(None, r, w, *a.values()))


OK = [{}, {"dtype": px.F32}, {"ldc": 7}, {"c": A + 2}, {"rows": {"k": 16}, "weights": {"k": 16}},
      {"weights": {"scales": A + 4}}, {"rows": {"ld": 160, "lds": 8}},
      {"rows": {"rows": 100_000, "k": 16384}, "weights": {"n": 4096, "k": 16384}}]
BAD = [{"dtype": 2}, {"dtype": -1}, {"c": 0}, {"c": A + 1}, {"dtype": px.F32, "c": A + 2}, {"ldc": 4},
       {"ldc": -5}, {"ldc": BIG}, {"rows": "none"}, {"weights": "none"}, {"weights": {"n": 0}},
       {"weights": {"n": -1}}, {"weights": {"n": 1 << 31}}, {"weights": {"k": 128}},
       {"weights": {"codes": 0}}, {"weights": {"scales": 0}}, {"weights": {"codes": A + 8}},
       {"weights": {"scales": A + 2}}, {"rows": {"k": 0}, "weights": {"k": 0}},
       {"rows": {"k": 136}, "weights": {"k": 136}},
       {"rows": {"k": (1 << 22) + 16}, "weights": {"k": (1 << 22) + 16}}, *({"rows": x} for x in BAD_ROWS)]


@pytest.mark.parametrize("ok", OK)
def test_gemm_takes(ok):
    assert _gemm(**{k: v for k, v in ok.items() if k != "order"}) == px.PHX_E_NOT_INIT
    assert _grouped(**ok) == px.PHX_E_NOT_INIT


@pytest.mark.parametrize("bad", BAD)
def test_gemm_refuses(bad):
    assert _gemm(**bad) == px.PHX_E_INVALID
    assert "gemm_f8" in px.lib().phx_last_error().decode()
    assert _grouped(**bad) == px.PHX_E_INVALID
    assert "gemm_f8_grouped" in px.lib().phx_last_error().decode()


def test_what_only_the_dense_product_refuses():
    assert _gemm(weights={"experts": 2}) == px.PHX_E_INVALID
    none = dict(codes=0, scales=0)
    assert _gemm({"rows": 0, **none}, none, c=0) == px.PHX_E_NOT_INIT
    assert _gemm({"rows": (1 << 31) - 1}, {"n": (1 << 31) - 1}) == px.PHX_E_INVALID
    assert "too large" in px.lib().phx_last_error().decode()


@pytest.mark.parametrize("ok", [{"order": 0, "M": 3}, {"M": 100}, {"order": 0, "M": 0},
                                {"rows": {"rows": (1 << 24) - 1, "k": 128}, "weights": {"k": 128}},
                                {"rows": {"rows": 1 << 24}, "order": 0},
                                {"weights": {"experts": 1}}, {"weights": {"experts": 65535}},
                                {"M": 0, "starts": 0, "order": 0, "c": 0}])
def test_grouped_takes(ok):
    assert _grouped(**ok) == px.PHX_E_NOT_INIT


@pytest.mark.parametrize("bad", [
    {"starts": 0}, {"starts": A + 2}, {"order": A + 1}, {"M": -1}, {"M": 1 << 31}, {"order": 0, "M": 4},
    {"rows": {"rows": 1 << 24}}, {"rows": {"rows": 1 << 20, "ld": 2048}}, {"rows": {"rows": 1 << 20, "lds": 512}},
    {"weights": {"experts": 0}}, {"weights": {"experts": -3}}, {"weights": {"experts": 65536}},
    {"M": (1 << 31) - 1, "weights": {"n": (1 << 31) - 1}}])
def test_grouped_refuses(bad):
    assert _grouped(**bad) == px.PHX_E_INVALID
    assert "gemm_f8_grouped" in px.lib().phx_last_error().decode()


# ---------------------------------------------------------------- the host's quantiser
@pytest.mark.parametrize("shape", [(1, 16), (128, 128), (130, 400), (2, 3, 200, 272)])
def test_f8_quantize(shape):
    rng = np.random.default_rng(len(shape))
    w = rng.standard_normal(shape) * 10.0 ** rng.uniform(-3, 3, (*shape[:-1], 1))
    w[..., 0, :5] = 0
    codes, scales = px.f8_quantize(w)
    N, K = shape[-2:]
    assert codes.shape == shape and codes.dtype == np.uint8
    assert scales.shape == (*shape[:-2], -(-N // 128), -(-K // 128)) and scales.dtype == np.float32
    for at in np.ndindex(shape[:-2]):
        for n in range(0, N, 128):
            for k in range(0, K, 128):
                b = w[at][n:n + 128, k:k + 128]
                a = np.abs(b).max()
                assert scales[at][n // 128, k // 128] == np.float32(a / 448)
                assert np.array_equal(codes[at][n:n + 128, k:k + 128], f8.codes_of(b * 448 / a))


def test_f8_quantize_of_zeros_and_what_it_refuses():
    codes, scales = px.f8_quantize(np.zeros((3, 160)))
    assert (codes & 127 == 0).all() and (scales == 0).all()
    for bad in (np.nan, np.inf, -np.inf, 1e300, 1e-40):
        w = np.zeros((4, 16))
        w[1, 2] = bad
        assert _rc(lambda: px.f8_quantize(w)) == px.PHX_E_INVALID
    for bad in (np.zeros(16), np.zeros((0, 16)), 3.0):
        assert _rc(lambda: px.f8_quantize(bad)) == px.PHX_E_INVALID


# ---------------------------------------------------------------- buffers that are too small
def _buffer(nbytes):
    b = px.DeviceBuffer.__new__(px.DeviceBuffer)
    b.nbytes, b.ptr = nbytes, A
    return b


@pytest.mark.parametrize("which,bytes_", [("x", 2 * (2 * 152 + 144)), ("r", 2 * 3 * 144), ("gain", 288),
                                          ("h", 2 * 3 * 144), ("y", 2 * 3 * 144)])
def test_norm_looks_at_its_buffers(which, bytes_):
    assert _norm(**{which: _buffer(bytes_), "ldx": 152}) == px.PHX_E_NOT_INIT
    with pytest.raises(px.PhxError, match="buffer holds"):
        px.launch_norm_f8(None, px.F16, *(_buffer(bytes_ - 1) if n == which else A
                                          for n in ("x", "r", "gain", "h", "y")), _rows(), 3, 144, 1e-5, 152)


def test_the_others_look_at_theirs():
    r, w = _rows(), _weights(experts=4)
    one = _weights()
    for good, call in [(2 * 3 * 288, lambda b: px.launch_glu_f8(None, px.F16, b, r)),
                       (4 * (2 * 9 + 5), lambda b: px.launch_gemm_f8(None, r, one, px.F32, b, ldc=9)),
                       (2 * 7 * 5, lambda b: px.launch_gemm_f8_grouped(None, r, w, A, A, 7, px.F16, b)),
                       (20, lambda b: px.launch_gemm_f8_grouped(None, r, w, b, A, 7, px.F16, A)),
                       (28, lambda b: px.launch_gemm_f8_grouped(None, r, w, A, b, 7, px.F16, A))]:
        assert _rc(lambda: call(_buffer(good))) == px.PHX_E_NOT_INIT
        with pytest.raises(px.PhxError, match="buffer holds"):
            call(_buffer(good - 1))
