"""The operators over 8-bit rows and weights together, as a program uses them: two
feed-forward layers on one stream, the first dense and the second of experts, each
the norm with the residual, the gate and value product, the activation, the
product back.  Every step is checked against 64 bits on the values that went into
it; then the whole is captured and replayed with other rows, routes and counts."""
import numpy as np
import pytest

import f8_model as f8
from hip_graph import Graph
from test_gpu_gemm_f8 import _bound

pytestmark = pytest.mark.gpu

WIDTH, INNER, EXPERTS, TOP = 272, 400, 5, 2


class Linear:
    def __init__(self, px, rng, K, N, experts=1):
        codes, scales = px.f8_quantize(rng.standard_normal((experts, N, K)) / K ** 0.5)
        self.bufs = [px.DeviceBuffer.from_array(x) for x in (codes, scales)]
        self.desc = px.F8Weights(*(b.ptr for b in self.bufs), experts, N, K)
        self.values = f8.weight_values(codes, scales)


class Rows:
    def __init__(self, px, M, K):
        self.shape, self.lds = (M, K), -(-K // 512) * 4
        self.codes, self.scales = px.DeviceBuffer(M * K), px.DeviceBuffer(4 * M * self.lds)
        self.desc = px.F8Rows(self.codes.ptr, self.scales.ptr, M, K)

    def get(self):
        return (self.codes.download(np.uint8, self.shape),
                self.scales.download(np.float32, (self.shape[0], self.lds))[:, :-(-self.shape[1] // 128)])

    def values(self):
        return f8.row_values(*self.get())


class Program:
    """M tokens: x += dense(norm(x)); y = experts(norm(x)), a row per token and choice."""

    def __init__(self, px, stream, M):
        self.px, self.s, self.M = px, stream, M
        self.rng = rng = np.random.default_rng(M)
        self.up, self.down = Linear(px, rng, WIDTH, 2 * INNER), Linear(px, rng, INNER, WIDTH)
        self.eup = Linear(px, rng, WIDTH, 2 * INNER, EXPERTS)
        self.edown = Linear(px, rng, INNER, WIDTH, EXPERTS)
        self.gain = [(1 + 0.1 * rng.standard_normal(WIDTH)).astype(np.float16) for _ in range(2)]
        self.dgain = [px.DeviceBuffer.from_array(g) for g in self.gain]
        R = M * TOP
        self.x, self.h = px.DeviceBuffer(2 * M * WIDTH), px.DeviceBuffer(2 * M * WIDTH)
        self.f = px.DeviceBuffer(2 * M * WIDTH)
        self.q, self.q2 = Rows(px, M, WIDTH), Rows(px, M, WIDTH)
        self.u, self.a = px.DeviceBuffer(2 * M * 2 * INNER), Rows(px, M, INNER)
        self.eu, self.ea = px.DeviceBuffer(2 * R * 2 * INNER), Rows(px, R, INNER)
        self.y = px.DeviceBuffer(4 * R * WIDTH)
        self.starts, self.order = px.DeviceBuffer(4 * (EXPERTS + 1)), px.DeviceBuffer(4 * R)

    def inputs(self, left=0):
        """Tokens, and each one's experts: the rows sorted by expert, the last `left`
        of them in no group."""
        M, R = self.M, self.M * TOP
        choice = np.stack([self.rng.permutation(EXPERTS)[:TOP] for _ in range(M)])
        choice[choice == 3] = 1  # an expert without rows
        order = np.argsort(choice.ravel(), kind="stable")
        starts = np.searchsorted(choice.ravel()[order], np.arange(EXPERTS + 1))
        self.h_starts, self.h_order = np.minimum(starts, R - left), order // TOP
        self.h_x, self.h_f = (self.rng.standard_normal((M, WIDTH)).astype(np.float16) for _ in range(2))
        for buf, v in ((self.x, self.h_x), (self.f, self.h_f), (self.starts, self.h_starts.astype(np.int32)),
                       (self.order, self.h_order.astype(np.int32)),
                       (self.y, np.full((R, WIDTH), 7, np.float32))):
            buf.upload(v)

    def launch(self):
        px, s, M, R = self.px, self.s, self.M, self.M * TOP
        # (what the layer before left in f is the residual)
        px.launch_norm_f8(s, px.F16, self.x, self.f, self.dgain[0], self.x, 0, self.q.desc, M, WIDTH, 1e-5)
        px.launch_gemm_f8(s, self.q.desc, self.up.desc, px.F16, self.u)
        px.launch_glu_f8(s, px.F16, self.u, self.a.desc)
        px.launch_gemm_f8(s, self.a.desc, self.down.desc, px.F16, self.x, 1.0, 1.0)
        px.launch_norm_f8(s, px.F16, self.x, 0, self.dgain[1], 0, self.h, self.q2.desc, M, WIDTH, 1e-5)
        px.launch_gemm_f8_grouped(s, self.q2.desc, self.eup.desc, self.starts, self.order, R, px.F16, self.eu)
        px.launch_glu_f8(s, px.F16, self.eu, self.ea.desc)
        px.launch_gemm_f8_grouped(s, self.ea.desc, self.edown.desc, self.starts, 0, R, px.F32, self.y)

    def check(self):
        M, R = self.M, self.M * TOP
        x = self.x.download(np.float16, (M, WIDTH))
        h, t, _ = f8.norm(self.h_x, self.h_f, self.gain[0], 1e-5)
        assert np.array_equal(self.q.get()[0], f8.codes_of(f8.quotients(t)[0]))
        u = self.u.download(np.float16, (M, 2 * INNER))
        a = self.q.values()
        want = a @ self.up.values[0].T
        assert (np.abs(u - want) <= _bound(want, a, self.up.values[0], np.float16)).all()
        self._glu(u, self.a)
        a, h = self.a.values(), h.astype(np.float64)
        want = a @ self.down.values[0].T + h
        assert (np.abs(x - want) <= _bound(want, a, self.down.values[0], np.float16, 1.0, np.abs(h))).all()
        _, t, factor = f8.norm(x, None, self.gain[1], 1e-5)
        assert np.array_equal(self.q2.get()[0], f8.codes_of(f8.quotients(t)[0]))
        y = t * factor
        assert (np.abs(self.h.download(np.float16, (M, WIDTH)) - y) <=
                np.abs(y) * (2.0 ** -11 + 2.0 ** -22) + 2.0 ** -24).all()
        eu, a = self.eu.download(np.float16, (R, 2 * INNER)), self.q2.values()
        got = self.y.download(np.float32, (R, WIDTH))
        for e in range(EXPERTS):
            b, end = self.h_starts[e:e + 2]
            rows = a[self.h_order[b:end]]
            want = rows @ self.eup.values[e].T
            assert (np.abs(eu[b:end] - want) <= _bound(want, rows, self.eup.values[e], np.float16)).all()
        b = self.h_starts[-1]
        self._glu(eu[:b], self.ea, b)
        ea = self.ea.values()
        for e in range(EXPERTS):
            b, end = self.h_starts[e:e + 2]
            want = ea[b:end] @ self.edown.values[e].T
            assert (np.abs(got[b:end] - want) <=
                    _bound(want, ea[b:end], self.edown.values[e], np.float32)).all()
        assert (got[self.h_starts[-1]:] == 7).all()  # rows in no group
        return x, got

    @staticmethod
    def _glu(u, rows, n=None):
        gate, value = np.split(u.astype(np.float64), 2, 1)
        q, a = f8.quotients(gate / (1 + np.exp(-gate)) * value)
        codes, scales = (v[:n] for v in rows.get())
        near = [f8.codes_of(np.clip(q * (1 + d), -448, 448)) for d in (-2.0 ** -19, 2.0 ** -19)]
        assert ((codes == near[0]) | (codes == near[1])).all()
        assert (np.abs(scales - a / 448) <= a / 448 * (2.0 ** -20 + 2.0 ** -23)).all()


@pytest.mark.parametrize("M,left", [(1, 0), (7, 3), (70, 0), (300, 40)])
def test_two_layers(px_gpu, stream, M, left):
    p = Program(px_gpu, stream, M)
    p.inputs(left)
    p.eu.zero(stream)  # rows in no group are read by the activation
    p.launch()
    stream.synchronize()
    p.check()


def test_captured_and_replayed(px_gpu):
    px = px_gpu
    s = px.Stream()
    p = Program(px, s, 33)
    p.inputs()
    p.eu.zero(s)
    p.launch()
    s.synchronize()
    g = Graph(s, p.launch)
    for left in (0, 5, 66, 1):
        p.inputs(left)
        g.replay()
        s.synchronize()
        x, y = p.check()
        p.x.upload(p.h_x)
        p.y.upload(np.full(y.shape, 7, np.float32))
        p.launch()
        s.synchronize()
        assert np.array_equal(p.x.download(np.float16, x.shape), x)
        assert np.array_equal(p.y.download(np.float32, y.shape), y)
    g.destroy()
    s.destroy()


def test_two_streams_at_once(px_gpu):
    # two programs, their launches by turns on two streams
    px = px_gpu
    programs = [Program(px, px.Stream(), M) for M in (40, 41)]
    for p in programs:
        p.inputs(2)
        p.eu.zero(p.s)
        p.s.synchronize()
    for _ in range(5):
        for p in programs:
            p.x.upload(p.h_x)
        for p in programs:
            p.launch()
    for p in programs:
        p.s.synchronize()
        p.check()
        p.s.destroy()
