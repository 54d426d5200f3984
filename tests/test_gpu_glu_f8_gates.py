"""phx_glu_f8 where e^-gate or gate / (1 + e^-gate) leaves f32 and the product with the
value does not: gates far below zero and next to it.  Values are within 2^-20 of the
formula's in 64 bits, so codes are those of a quotient within 2^-19 and scales within
2^-20 and their own rounding, 2^-24; where f32 has subnormal numbers, within one of them."""
import numpy as np
import pytest

import f8_model as f8
from test_gpu_f8_rows import _glu, _glu_values

pytestmark = pytest.mark.gpu

FAR = [-79.5, -80.0, -80.5, -85.0, -87.0, -88.0, -88.5, -88.72, -88.75, -89.0, -90.0, -93.0, -96.0, -99.0]
FURTHER = [-101.0, -110.0, -150.0, -200.0, -260.0]  # with large f32 values only


def _check(codes, scales, u):
    v = _glu_values(u)
    # (the values are f32: of the gates listed here -200 and -260 give at most 200 e^-200 3e37 =
    # 8.3e-48, below half of the smallest f32, 2^-150 = 7.0e-46, so zeros)
    v = np.where(np.abs(v) < 2.0 ** -126, v.astype(np.float32), v)
    q, a = f8.quotients(v)
    lo, hi = (f8.codes_of(np.clip(q * (1 + d), -448, 448)) for d in (-2.0 ** -19, 2.0 ** -19))
    assert ((codes == lo) | (codes == hi)).all()
    want = a / 448
    assert (np.abs(scales - want) <= want * (2.0 ** -20 + 2.0 ** -23) + 2.0 ** -149).all()


def _type(bits):
    return np.float16 if bits == 16 else np.float32


def _value(bits):
    return 60000.0 if bits == 16 else 3e37


@pytest.mark.parametrize("bits", [16, 32])
def test_one_gate_a_block(px_gpu, stream, bits):
    g = np.array(FAR + (FURTHER if bits == 32 else []))
    u = np.zeros((g.size, 256), _type(bits))
    u[:, 77], u[:, 128 + 77] = g, _value(bits)
    _check(*_glu(px_gpu, stream, bits, u), u)


@pytest.mark.parametrize("bits", [16, 32])
def test_blocks_of_far_gates(px_gpu, stream, bits):
    # every lane on either side of the border, results of one size
    rng = np.random.default_rng(bits)
    t = _type(bits)
    g = rng.uniform(-93, -78, (40, 272)).astype(t)
    e = np.exp(-80 - g.astype(np.float64))
    value = rng.uniform(0.5, 1, g.shape) * rng.choice([-1, 1], g.shape)
    value = (value * e * 1e5).clip(-6e4, 6e4) if bits == 16 else value * e * 1e30
    u = np.concatenate([g, value.astype(t)], 1)
    _check(*_glu(px_gpu, stream, bits, u), u)


def test_far_gates_with_large_values(px_gpu, stream):
    rng = np.random.default_rng(7)
    g = rng.uniform(-150, -60, (60, 400)).astype(np.float32)
    value = (rng.uniform(0.5, 1, g.shape) * np.exp(-70 - g.astype(np.float64))).astype(np.float32)
    u = np.concatenate([g, value], 1)
    _check(*_glu(px_gpu, stream, 32, u), u)


@pytest.mark.parametrize("bits", [16, 32])
def test_a_far_gate_changes_no_neighbour(px_gpu, stream, bits):
    rng = np.random.default_rng(9)
    u = (rng.standard_normal((60, 2 * 272)) * 4).astype(_type(bits))
    clean = _glu(px_gpu, stream, bits, u)
    most = np.finfo(_type(bits)).min
    far = u.copy()
    at = rng.integers(0, 272, (60, 9))
    # (not the largest of their block, which the scale goes by)
    v = np.abs(f8.blocks_of(_glu_values(u)))
    for m in range(60):
        for k in at[m]:
            if v[m, k // 128, k % 128] < v[m, k // 128].max():
                far[m, k] = rng.choice([-80.5, -95, -1e4, most])
    codes, scales = _glu(px_gpu, stream, bits, far)
    moved = far[:, :272] != u[:, :272]
    assert moved.sum() > 400
    assert np.array_equal(codes[~moved], clean[0][~moved]) and np.array_equal(scales, clean[1])
    assert (codes[moved] & 127 == 0).all()
    _check(codes, scales, far)


@pytest.mark.parametrize("bits", [16, 32])
def test_the_lowest_gates(px_gpu, stream, bits):
    # zeros with the sign of the product; an infinite gate is no number
    t = _type(bits)
    u = np.zeros((4, 256), t)
    u[0, 5], u[0, 133] = np.finfo(t).min, np.finfo(t).max
    u[1, 5], u[1, 133] = np.finfo(t).min, -1
    u[2, 5], u[2, 133] = -np.inf, 1
    u[3, 5], u[3, 133] = -np.inf, 0
    codes, scales = _glu(px_gpu, stream, bits, u)
    assert (codes[:2] & 127 == 0).all() and (scales[:2] == 0).all()
    assert codes[0, 5] == 0x80 and codes[1, 5] == 0
    assert np.isnan(f8.VALUES[codes[2:]]).all() and np.isnan(scales[2:]).all()


def test_gates_next_to_zero(px_gpu, stream):
    # half of a subnormal gate has fewer bits than the gate
    g = np.array([1, 3, 5, -7, 1001, -(1 << 22) - 1, (1 << 23) - 1, (1 << 23) + 1, -(1 << 24) - 3])
    g = np.concatenate([np.ldexp(g.astype(np.float64), -149), [2.0 ** -124, -2.0 ** -100]])
    for value in (3e38, -2.0 ** 100, 2.0 ** 30):
        u = np.zeros((g.size, 256), np.float32)
        u[:, 9], u[:, 137] = g, value
        _check(*_glu(px_gpu, stream, 32, u), u)
    rng = np.random.default_rng(3)
    g = np.ldexp(rng.integers(-4000, 4000, (30, 272)).astype(np.float64), -149).astype(np.float32)
    u = np.concatenate([g, (rng.standard_normal(g.shape) * 1e37).astype(np.float32)], 1)
    _check(*_glu(px_gpu, stream, 32, u), u)
