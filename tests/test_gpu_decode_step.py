"""The decode operators together, as a program that answers with a model uses
them: two layers of 4-bit projections and cached attention, a prompt in chunks,
sequences forked and compacted between steps, all on one stream.  Every step is
checked against 64 bits on the values that went into it."""
import numpy as np
import pytest

from kv4_model import Pool, attention, quantise

pytestmark = pytest.mark.gpu

H, R, D, P, WIDTH, LAYERS, PAGES, GROUP = 2, 3, 64, 32, 200, 2, 16, 64
HQ = H * R


class Linear:
    def __init__(self, px, stream, rng, K, N):
        self.px, self.K, self.N = px, K, N
        codes, self.scales, zeros = px.w4_quantize(rng.standard_normal((K, N)) / K ** 0.5, GROUP)
        g = np.arange(K) // GROUP
        self.w = (codes.astype(np.int64) - zeros[g]) * self.scales.astype(np.float64)[g]
        self.bufs = [px.DeviceBuffer(px.w4_packed_bytes(N, K)),
                     px.DeviceBuffer.from_array(self.scales), px.DeviceBuffer.from_array(zeros)]
        raw = px.DeviceBuffer.from_array(codes)
        px.w4_pack(stream, raw, self.bufs[0], N, K)
        stream.synchronize()

    def __call__(self, stream, x, M, out, beta=0.0, rows=None):
        """Rows in launches of 64, onto out (kept with beta 1)."""
        px = self.px
        for r in range(0, M, 64):
            px.launch_gemv_w4(stream, px.F16, x.ptr + 2 * r * self.K, *self.bufs,
                              out.ptr + 2 * r * self.N, min(64, M - r), self.N, self.K, GROUP, 1.0,
                              beta)

    def check(self, x, got, base=0):
        x = x.astype(np.float64)
        want, mag = x @ self.w + base, np.abs(x) @ np.abs(self.w) + np.abs(base)
        inner = (self.K + 8) * mag * 2.0 ** -24
        assert (np.abs(got - want) <= np.abs(want) * 2.0 ** -11 + 1.001 * inner + 2.0 ** -25).all()


class Program:
    def __init__(self, px, stream):
        self.px, self.stream, rng = px, stream, np.random.default_rng(42)
        self.rng, self.pages = rng, px.Pages(PAGES, P)
        self.page_bytes = px.kv4_page_bytes(H, D, P)
        self.model = [Pool(PAGES, H, D, P) for _ in range(LAYERS)]
        self.pool = px.DeviceBuffer.from_array(np.stack([m.data for m in self.model]))
        self.stride = PAGES * self.page_bytes
        sizes = [(WIDTH, HQ * D), (WIDTH, H * D), (WIDTH, H * D), (HQ * D, WIDTH)]
        self.layers = [[Linear(px, stream, rng, *s) for s in sizes] for _ in range(LAYERS)]

    def apply(self):
        src, dst = self.pages.pending()
        for m in self.model:
            m.data[dst] = m.data[src]
        self.pages.apply(self.stream, self.pool, self.page_bytes, LAYERS, self.stride)

    def step(self, seqs, counts, x):
        """New rows x [sum(counts), WIDTH] of these sequences through the layers."""
        px, s = self.px, self.stream
        lens = np.zeros(len(seqs), np.int32)
        tables = []
        for i, (seq, n) in enumerate(zip(seqs, counts)):
            lens[i] = self.length[seq] = self.length[seq] + n
            self.pages.resize(seq, self.length[seq])
        tables = [self.pages.table(seq) for seq in seqs]
        self.apply()
        stride = max(len(t) for t in tables)
        table = np.full((len(seqs), stride), -1, np.int32)
        for row, t in zip(table, tables):
            row[:len(t)] = t
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        M = int(starts[-1])
        d = [px.DeviceBuffer.from_array(a) for a in (table, lens, starts)]
        batch = px.Kv4Batch(d[0].ptr, stride, d[1].ptr, d[2].ptr, len(seqs), max(counts),
                            int(lens.max()), M)
        dx = px.DeviceBuffer.from_array(x)
        dq, dk, dv, do = (px.DeviceBuffer(2 * M * n * D) for n in (HQ, H, H, HQ))
        for layer in range(LAYERS):
            q, k, v, o = self.layers[layer]
            cache = px.Kv4Cache(self.pool.ptr + layer * self.stride, PAGES, H, D, P)
            for lin, out in ((q, dq), (k, dk), (v, dv)):
                lin(s, dx, M, out)
            px.launch_kv4_append(s, cache, batch, px.F16, dk, dv)
            px.launch_kv4_attention(s, cache, batch, px.F16, dq, do, HQ, D ** -0.5, True)
            o(s, do, M, dx, beta=1.0)  # the residual
            s.synchronize()
            hq, hk, hv, ho = (b.download(np.float16, (M, n, D))
                              for b, n in ((dq, HQ), (dk, H), (dv, H), (do, HQ)))
            for lin, got in ((q, hq), (k, hk), (v, hv)):
                lin.check(x, got.reshape(M, -1))
            m = self.model[layer]
            for i in range(len(seqs)):
                for r in range(counts[i]):
                    pos = lens[i] - counts[i] + r
                    for h in range(H):
                        for is_v, rows in ((False, hk), (True, hv)):
                            m.write(table[i, pos // P], h, pos % P, is_v,
                                    *quantise(rows[starts[i] + r, h]))
            want, seen, off = attention(m, table, lens, starts, max(counts), int(lens.max()), hq,
                                        D ** -0.5, True)
            assert seen.all()
            assert (np.abs(ho - want) <= np.abs(want) * 2.0 ** -11 + 1.001 * off + 2.0 ** -25).all()
            new = dx.download(np.float16, x.shape)
            o.check(ho.reshape(M, -1), new, x.astype(np.float64))
            x = new
        got = self.pool.download(np.uint8, (LAYERS, *self.model[0].data.shape))
        assert np.array_equal(got, np.stack([m.data for m in self.model]))
        return x

    length = None


def test_prompt_forks_steps_and_compaction(px_gpu, stream):
    p = Program(px_gpu, stream)
    p.length = {}

    def rows(n):
        return p.rng.standard_normal((n, WIDTH)).astype(np.float16)

    a, b = p.pages.new(), p.pages.new()
    p.length = {a: 0, b: 0}
    p.step([a, b], [70, 5], rows(75))  # prompts, more rows than one product takes
    c = p.pages.fork(a)
    p.length[c] = p.length[a]
    p.step([a, b, c], [1, 1, 1], rows(3))  # the fork's last page is copied
    assert len(set(p.pages.table(a)) & set(p.pages.table(c))) == 2
    p.step([c, b, a], [1, 30, 2], rows(33))  # a chunk and tokens in one call
    p.pages.free(a)
    d = p.pages.fork(c)
    p.length[d] = p.length[c]
    p.pages.compact()
    p.apply()
    assert p.pages.stats()[0] == p.pages.stats()[1]
    p.step([d, c, b], [2, 1, 1], rows(4))
    p.pages.resize(d, 40)  # a sequence cut back, and on from there
    p.length[d] = 40
    p.step([b, d], [1, 1], rows(2))
