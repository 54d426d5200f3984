"""How far f32 attention over the 4-bit cache is off on ordinary inputs: the
error's norm against the output's.  (The bounds of test_gpu_kv4.py are worst
cases, 1000 times and more of this; queries or weights that lost their second
f16 term would stay within them.)

The tolerance, from the arithmetic the header states.  Inputs: values of mean
zero, scores whose parts are below 8 in log2 units, up to 64 steps a wave.  An
output is a weighted mean of the values, so an error e_j of each weight for
itself, relative, leaves the output as far off as its own norm times the
rms of e_j.  In units of 2^-21 the parts of that are
  the score  8 sums that may cut what is below their last bit, 2^-21 of values
             in 4 .. 8, rms 2^-21/sqrt 3 each, and 3 rounded operations, of half
             as much: sqrt(8/3 + 3/12), times ln 2                      1.18
  exp2 and the weight's two f16 terms, 2^-23 each                       0.2
  the weights' sum, 64 roundings of 2^-24                               0.58
  the product with the values, 64 steps of two sums cut at 2^-23        1.63
together 2.1 * 2^-21 = 1.0e-6: the tolerance is 2^-19, twice that.  A single
f16 term is off by up to 2^-12 of the value, rms about 2^-13: 60 tolerances of
a score of size 1."""
import numpy as np
import pytest

from kv4_model import attention
from test_gpu_kv4 import Call, any_stream  # noqa: F401

TOLERANCE = 2.0 ** -19

# (heads, query heads per head, page, lens, starts, max_q): 4, 8, 16 and 32
# columns a workgroup, in the wide forms or split where the keys are many, and
# whole workgroups of columns
SHORT = [60, 130, 33, 257, 96, 1, 64, 200]
CASES = [(2, 4, 64, [1500, 700], None, 1), (1, 3, 32, [4000], None, 1), (2, 8, 64, [1300, 90], None, 1),
         (1, 16, 128, [2100], None, 1), (2, 4, 64, [900, 400], None, 6),
         (2, 4, 64, [500, 300], None, 1), (2, 7, 64, [500], None, 1), (1, 16, 64, [600, 601], None, 1),
         (4, 6, 32, SHORT * 5, np.arange(41) * 2, 13), (4, 33, 64, SHORT * 5, None, 3)]


def _fill(c):
    """Codes of every kind; values about 0, a scale of its own for each token."""
    p, r = c.pool, c.rng
    P, D = p.P, p.D
    p.data[:, :, :P * D] = r.integers(0, 256, (p.pages, p.heads, P * D))
    par = np.empty((p.pages, p.heads, 2, P, 2), np.float16)
    par[..., 0] = r.uniform(0.05, 0.2, par.shape[:-1])
    par[..., 1] = -7.5 * par[..., 0].astype(np.float64) + r.uniform(-0.05, 0.05, par.shape[:-1])
    p.data[:, :, P * D:] = par.reshape(p.pages, p.heads, -1).view(np.uint8)
    return c


def _relative(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_error_of_f32_attention(px_gpu, any_stream, D, case):  # noqa: F811
    heads, R, P, lens, starts, max_q = CASES[case]
    c = _fill(Call(px_gpu, heads, D, P, lens, starts, max_q, seed=case)).upload()
    q = c.rng.standard_normal((c.rows, heads * R, D)).astype(np.float32)
    want, seen, _ = attention(c.pool, c.table, c.lens, c.starts, max_q, c.max_len, q, D ** -0.5, True)
    got = c.attend(any_stream, 32, q, D ** -0.5).astype(np.float64)
    assert _relative(got[seen], want[seen]) <= TOLERANCE


def _two(x):
    hi = x.astype(np.float16)
    return hi.astype(np.float64) + (x - hi).astype(np.float16)


def _one(x):
    return x.astype(np.float16).astype(np.float64)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 20, 1500])
def test_a_lost_term_is_past_the_tolerance(D, n):
    """The same inputs in 64 bits but for the queries or the weights."""
    r = np.random.default_rng(n)
    size = r.uniform(0.05, 0.2, (2, n, 1))
    k, v = size * (r.integers(0, 16, (2, n, D)) - 7.5) + r.uniform(-0.05, 0.05, (2, n, 1))
    q = r.standard_normal((8, D))

    def run(queries, weights):
        t = queries(q * 2.0 ** 8) @ k.T * (D ** -0.5 * np.log2(np.e) * 2.0 ** -8)
        assert np.abs(t).max() < 8
        w = 2.0 ** (t - t.max(-1, keepdims=True) + 7)
        return weights(w * size[1, :, 0]) @ (v / size[1]) / w.sum(-1, keepdims=True)

    same = lambda x: x  # noqa: E731
    want = run(same, same)
    assert _relative(run(_two, _two), want) < TOLERANCE / 8
    if n > 1:  # of one key the weight is 1, whatever the score
        assert _relative(run(_one, _two), want) > 8 * TOLERANCE
    assert _relative(run(_two, _one), want) > 8 * TOLERANCE
