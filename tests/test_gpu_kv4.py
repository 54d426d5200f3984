"""The 4-bit cache on the GPU: append bit for bit, read, and attention within
the bounds of its arithmetic, against tests/kv4_model.py (64 bits)."""
import os
import subprocess
import sys

import numpy as np
import pytest

from hip_graph import Graph
from kv4_model import Pool, attention, page_of, quantise, rows_of

pytestmark = pytest.mark.gpu


def _t(bits):
    return np.float16 if bits == 16 else np.float32


class Call:
    """A pool and the sequences of a call, on the host and on the GPU."""

    def __init__(self, px, heads, D, P, lens, starts=None, max_q=1, max_len=None, rows=None,
                 seed=0, spare=2, stride=None):
        self.px, self.rng = px, np.random.default_rng(seed)
        self.lens = np.asarray(lens, np.int32)
        self.starts = None if starts is None else np.asarray(starts, np.int32)
        self.max_q = max_q
        most = max(int(self.lens.max(initial=0)), 1)
        self.stride = stride if stride is not None else -(-most // P)
        self.max_len = most if max_len is None else max_len
        B = len(self.lens)
        self.rows = rows if rows is not None else (B * max_q if starts is None else int(starts[-1]))
        pages = B * self.stride + spare
        self.table = self.rng.permutation(pages)[:B * self.stride].reshape(B, self.stride)
        self.table = self.table.astype(np.int32)
        self.pool = Pool(pages, heads, D, P)

    def fill(self, low=-1.0, width=2.0):
        """Random codes and parameters in every slot that holds a token; the
        others stay all ones (NaN)."""
        p, r = self.pool, self.rng
        for b, n in enumerate(self.lens):
            for t in range(min(int(n), self.stride * p.P)):
                page = page_of(p, self.table, b, t)
                if page < 0:
                    continue
                for h in range(p.heads):
                    for v in (False, True):
                        s = width / 15 * (0.3 + r.random())
                        p.write(page, h, t % p.P, v, r.integers(0, 16, p.D).astype(np.uint8), s,
                                low * (0.5 + r.random()))
        return self

    def upload(self):
        px, p = self.px, self.pool
        self.d_pool = px.DeviceBuffer.from_array(p.data)
        self.d = [px.DeviceBuffer.from_array(x) for x in (self.table, self.lens)]
        self.d_starts = None if self.starts is None else px.DeviceBuffer.from_array(self.starts)
        self.cache = px.Kv4Cache(self.d_pool.ptr, p.pages, p.heads, p.D, p.P)
        self.batch = px.Kv4Batch(self.d[0].ptr, self.stride, self.d[1].ptr,
                                 self.d_starts.ptr if self.d_starts else 0, len(self.lens),
                                 self.max_q, self.max_len, self.rows)
        return self

    def cap(self):
        return min(self.max_len, self.stride * self.pool.P)

    def mine(self):
        for b in range(len(self.lens)):
            yield b, *rows_of(b, self.lens, self.starts, self.max_q, self.rows, self.cap())

    def attend(self, stream, bits, q, scale=0.125, causal=True, pad=0, extra=0):
        """(O rows, device call's other memory intact) over q [rows, Hq, D]."""
        px, t = self.px, _t(bits)
        rows, Hq, D = q.shape
        ld = Hq * D + pad
        host = np.full((rows + extra, ld), np.nan, t)
        host[:rows, :Hq * D] = q.reshape(rows, -1)
        out = np.full((rows + extra, ld), 33, t)
        dq, do = px.DeviceBuffer.from_array(host), px.DeviceBuffer.from_array(out)
        px.launch_kv4_attention(stream, self.cache, self.batch, px.F16 if bits == 16 else px.F32,
                                dq, do, Hq, scale, causal, ld, ld)
        px.synchronize()
        got = do.download(t, out.shape)
        assert (got[rows:] == 33).all() and (got[:, Hq * D:] == 33).all(), "stored outside O"
        return got[:rows, :Hq * D].reshape(rows, Hq, D)

    def check(self, stream, bits, q, scale=0.125, causal=True, pad=0, extra=0):
        q = q.astype(_t(bits))
        want, seen, off = attention(self.pool, self.table, self.lens, self.starts, self.max_q,
                                    self.max_len, q, scale, causal)
        got = self.attend(stream, bits, q, scale, causal, pad, extra).astype(np.float64)
        half = np.finfo(_t(bits)).eps / 2
        tiny = 2.0 ** -25 if bits == 16 else 2.0 ** -149
        assert (got[~seen] == 33).all(), "a row outside the call was stored"
        err = np.abs(got - want)
        bound = (np.abs(want) + off) * half + off + tiny
        bad = ~(err <= bound) & seen[:, None, None]
        assert not bad.any(), (np.argwhere(bad)[:4], np.max(err[bad] / bound[bad]))
        return got


@pytest.fixture(params=["bound", "bare"])
def any_stream(request, px_gpu, stream):
    """The session's stream with a workspace, and one without."""
    if request.param == "bound":
        yield stream
    else:
        s = px_gpu.Stream()
        yield s
        s.destroy()


# ------------------------------------------------------------------ append
def _values(rng, rows, heads, D, t):
    """Rows of every kind: normal, constant, zeros, tiny, wide, one outlier,
    and values in the middle of two codes."""
    x = rng.standard_normal((rows, heads, D))
    kind = rng.integers(0, 8, (rows, heads))
    x[kind == 1] = 0.3
    x[kind == 2] = 0
    x[kind == 3] *= 2.0 ** -22
    x[kind == 4] *= 20000
    x[kind == 5, 3] = 900
    mid = kind == 6
    x[mid] = (rng.integers(0, 31, (mid.sum(), D)) / 2 - 4) * 0.25
    x[mid, 0], x[mid, 1] = -1, 2.75  # a range of 15 steps of 0.25
    x[kind == 7] = np.abs(x[kind == 7]) + 100
    return x.clip(-65000, 65000).astype(t)


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads,P,lens,starts,max_q", [
    (1, 32, [1], None, 1), (3, 32, [1, 32, 33, 0, 70], None, 1), (2, 64, [100, 7], None, 5),
    (2, 128, [40, 3, 129, 0, 300], [0, 1, 4, 44, 44, 51], 40), (5, 256, [300], None, 260),
    (2, 32, [5, 2], None, 9)])
def test_append_bit_for_bit(px_gpu, stream, bits, D, heads, P, lens, starts, max_q):
    px, t = px_gpu, _t(bits)
    c = Call(px, heads, D, P, lens, starts, max_q, seed=P + D).upload()
    pads = (8, 16)
    host = [np.full((c.rows, heads * D + pad), np.nan, t) for pad in pads]
    k, v = (_values(c.rng, c.rows, heads, D, t) for _ in pads)
    for h, x in zip(host, (k, v)):
        h[:, :heads * D] = x.reshape(c.rows, -1)
    dk, dv = (px.DeviceBuffer.from_array(h) for h in host)
    px.launch_kv4_append(stream, c.cache, c.batch, px.F16 if bits == 16 else px.F32, dk, dv,
                         *(heads * D + p for p in pads))
    for b, n, mine in c.mine():
        for row, pos in mine:
            if pos < 0:
                continue
            page = page_of(c.pool, c.table, b, pos)
            for h in range(heads):
                for is_v, x in ((False, k), (True, v)):
                    c.pool.write(page, h, pos % P, is_v, *quantise(x[row, h]))
    stream.synchronize()
    got = c.d_pool.download(np.uint8, c.pool.data.shape)
    assert np.array_equal(got, c.pool.data)
    # and what was stored is near what was given: half a step, the two f16
    # roundings of the parameters, and the steps below 2^-24
    for b, n, mine in c.mine():
        for row, pos in mine:
            if pos >= 0:
                for h in range(heads):
                    x = k[row, h].astype(np.float64)
                    got = c.pool.value(page_of(c.pool, c.table, b, pos), h, pos % P, False)
                    step = max((x.max() - x.min()) / 15, 2.0 ** -24)
                    slack = np.abs(x.min()) * 2.0 ** -11 + 15 * step * 2.0 ** -11 + 16 * 2.0 ** -25
                    assert np.abs(got - x).max() <= step / 2 + slack


@pytest.mark.parametrize("D", [64, 128])
def test_append_next_to_every_tie(px_gpu, stream, D):
    # f32 elements on ties between two codes and 1, 2 and 40 steps beside them,
    # and ranges whose f16 scale is such a tie or next to one
    px, heads, rows, P = px_gpu, 2, 300, 64
    c = Call(px, heads, D, P, [rows], None, rows, seed=1).upload()
    r = c.rng
    steps = np.array([-40, -2, -1, 0, 1, 2, 40])
    x = np.empty((2, rows, heads, D), np.float32)
    for i in np.ndindex(2, rows, heads):
        low = np.float64(np.float16(r.standard_normal() * 2.0 ** r.integers(-6, 6)))
        s = np.float64(np.float16(r.uniform(1, 2) * 2.0 ** r.integers(-8, 4)))
        tie = (low + s * (r.integers(0, 15, D) + 0.5)).astype(np.float32)
        row = (tie.view(np.int32) + r.choice(steps, D).astype(np.int32)).view(np.float32)
        row[0] = low
        # the largest: 15 scales, or 15 times the middle of two f16 and beside it
        mid = (s + np.float64(np.nextafter(np.float16(s), np.float16(np.inf)))) / 2
        row[1] = low + 15 * s if r.random() < 0.5 else \
            (np.float32(low + 15 * mid).view(np.int32) + np.int32(r.choice(steps))).view(np.float32)
        x[i] = np.clip(row, row[0], row[1])
    dk, dv = (px.DeviceBuffer.from_array(y.reshape(rows, -1)) for y in x)
    px.launch_kv4_append(stream, c.cache, c.batch, px.F32, dk, dv)
    stream.synchronize()
    got = Pool(c.pool.pages, heads, D, P)
    got.data = c.d_pool.download(np.uint8, c.pool.data.shape)
    checked = 0
    for row in range(rows):
        for h in range(heads):
            for v in (False, True):
                # a step below 0.0 is a NaN, which is no value to append
                if not np.isfinite(x[int(v), row, h]).all():
                    continue
                mine = got.raw(page_of(c.pool, c.table, 0, row), h, row % P, v)
                for y, z in zip(mine, quantise(x[int(v), row, h])):
                    assert np.array_equal(y, z), (row, h, v)
                checked += 1
    assert checked > 1100


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("D", [64, 128])
def test_append_and_read_skip_what_is_no_page(px_gpu, stream, bits, D):
    px, t = px_gpu, _t(bits)
    heads, P = 2, 32
    c = Call(px, heads, D, P, [70, 70, 1 << 30, -5], [3, 43, 80, 99, 101], 40, max_len=70, rows=100,
             stride=3)
    c.table[0, 1], c.table[1, 2], c.table[2, 1] = -1, c.pool.pages, 1 << 30
    c.upload()
    k, v = (c.rng.standard_normal((c.rows, heads, D)).astype(t) for _ in range(2))
    dk, dv = px.DeviceBuffer.from_array(k), px.DeviceBuffer.from_array(v)
    dtype = px.F16 if bits == 16 else px.F32
    px.launch_kv4_append(stream, c.cache, c.batch, dtype, dk, dv)
    back = np.full(k.shape, 5, t)
    bk, bv = px.DeviceBuffer.from_array(back), px.DeviceBuffer.from_array(back)
    px.launch_kv4_read(stream, c.cache, c.batch, dtype, bk, bv)
    want = [back.copy(), back.copy()]
    for b, n, mine in c.mine():
        for row, pos in mine:
            page = page_of(c.pool, c.table, b, pos) if pos >= 0 else -1
            for h in range(heads):
                for is_v, x in ((False, k), (True, v)):
                    if page >= 0:
                        c.pool.write(page, h, pos % P, is_v, *quantise(x[row, h]))
                    want[is_v][row, h] = 0 if page < 0 else _stands_for(c.pool, page, h, pos % P,
                                                                        is_v, t)
    stream.synchronize()
    assert np.array_equal(c.d_pool.download(np.uint8, c.pool.data.shape), c.pool.data)
    assert np.array_equal(bk.download(t, k.shape), want[0])
    assert np.array_equal(bv.download(t, k.shape), want[1])


def _stands_for(pool, page, h, slot, v, t):
    codes, s, m = pool.raw(page, h, slot, v)
    return (codes.astype(np.float32) * np.float32(s) + np.float32(m)).astype(t)


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("D,heads,R,P", [(64, 1, 1, 32), (64, 3, 4, 64), (128, 2, 8, 32),
                                         (128, 1, 16, 128), (64, 2, 20, 256), (128, 2, 5, 64)])
def test_one_token(px_gpu, any_stream, bits, D, heads, R, P):
    c = Call(px_gpu, heads, D, P, [1, 0, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 250, 600],
             seed=R).fill().upload()
    c.check(any_stream, bits, c.rng.standard_normal((c.rows, heads * R, D)), D ** -0.5)


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,heads,R,P,lens,starts,max_q", [
    (64, 1, 1, 32, [100], None, 7), (128, 2, 4, 64, [3, 70, 0, 40], None, 40),
    (64, 2, 3, 32, [200, 5, 33, 1], [0, 65, 70, 71, 72], 65), (128, 1, 8, 32, [150], None, 150),
    (64, 1, 16, 128, [90, 17], [2, 19, 19], 17), (128, 2, 2, 256, [300, 20], [0, 33, 40], 33)])
def test_chunks(px_gpu, any_stream, bits, causal, D, heads, R, P, lens, starts, max_q):
    c = Call(px_gpu, heads, D, P, lens, starts, max_q, seed=max_q).fill().upload()
    c.check(any_stream, bits, c.rng.standard_normal((c.rows, heads * R, D)), D ** -0.5, causal,
            pad=16, extra=3)


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths_tables_and_starts_that_lie(px_gpu, any_stream, bits, causal):
    # lengths past the table and below 0, entries that are no page, starts that
    # go backwards, past the rows and below 0
    heads, D, P = 2, 64, 32
    c = Call(px_gpu, heads, D, P, [1 << 30, -7, 90, 96, 64, 20, 96],
             [-3, 4, 4, 2, 12, 30, 26, 1 << 30], 20, max_len=90, rows=33, stride=3)
    c.table[0, 1], c.table[2, 0], c.table[3, :], c.table[4, 1] = -1, 1 << 30, -9, c.pool.pages
    c.lens[0] = 90  # to fill its slots
    c.fill()
    c.lens[0] = 1 << 30
    c.upload()
    q = c.rng.standard_normal((c.rows, heads * 3, D))
    got = c.attend(any_stream, bits, q.astype(_t(bits)), 0.125, causal)
    # rows that two sequences claim hold one of theirs; the others are checked
    claimed = np.zeros(c.rows, int)
    for b, n, mine in c.mine():
        for row, _ in mine:
            claimed[row] += 1
    want, seen, off = attention(c.pool, c.table, c.lens, c.starts, c.max_q, c.max_len,
                                q.astype(_t(bits)), 0.125, causal)
    once = claimed == 1
    assert once.sum() > 12 and (got[claimed == 0] == 33).all()
    half = np.finfo(_t(bits)).eps / 2
    assert (np.abs(got[once] - want[once]) <= (np.abs(want) + off)[once] * half + off[once]
            + 2.0 ** -25).all()


def test_no_pages_at_all(px_gpu, stream):
    c = Call(px_gpu, 1, 64, 32, [40], max_len=40).upload()
    c.batch.table, c.batch.table_stride = 0, 0
    assert (c.attend(stream, 16, np.ones((1, 2, 64), np.float16)) == 0).all()


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_that_rise_and_fall(px_gpu, any_stream, bits, D):
    # along the keys the scores rise by hundreds, fall again, and one key far
    # behind outweighs all: the running maximum has to follow
    c = Call(px_gpu, 2, D, 32, [700, 700, 700], seed=3).fill()
    p, r = c.pool, c.rng
    ramp = [np.linspace(-6, 6, 700), np.linspace(6, -6, 700), np.full(700, -3.0)]
    ramp[2][613] = 8
    for b in range(3):
        for t in range(700):
            for h in range(2):
                codes = r.integers(6, 9, D).astype(np.uint8)
                p.write(c.table[b, t // 32], h, t % 32, False, codes, 0.01, ramp[b][t])
    c.upload()
    q = np.abs(r.standard_normal((3, 4, D))) * np.array([1, -1])[r.integers(0, 2, (3, 4, 1))]
    c.check(any_stream, bits, q, 1.0)


@pytest.mark.parametrize("bits", [16, 32])
def test_scales_of_every_size(px_gpu, any_stream, bits):
    # V's scales from the smallest f16 to the largest, next to each other, with
    # scores that make up for them: weight times scale spans 80 powers of two
    D = 64
    c = Call(px_gpu, 1, D, 64, [500], seed=5).fill()
    p, r = c.pool, c.rng
    for t in range(500):
        e = int(r.integers(-24, 12))
        p.write(c.table[0, t // 64], 0, t % 64, True, r.integers(0, 16, D).astype(np.uint8),
                2.0 ** e, float(r.standard_normal()) * 2.0 ** min(e + 3, 14))
        p.write(c.table[0, t // 64], 0, t % 64, False, np.zeros(D, np.uint8), 2.0 ** -24,
                -e * 0.02)
    c.upload()
    c.check(any_stream, bits, np.ones((1, 3, D)) * np.array([0.5, 1, 2])[None, :, None], 1.0)


@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -8, 300.0, 60000.0])
def test_queries_of_every_size(px_gpu, any_stream, bits, size):
    c = Call(px_gpu, 1, 128, 32, [90, 33], seed=6).fill().upload()
    q = c.rng.uniform(-1, 1, (2, 4, 128)) * size
    q[0, 1] = 0
    q[1, 2, 5:] *= 2.0 ** -12
    c.check(any_stream, bits, q, 0.1 / size)


@pytest.mark.parametrize("scale", [0.0, -0.25, 4.0])
def test_any_scale(px_gpu, any_stream, scale):
    c = Call(px_gpu, 2, 64, 32, [130, 64], seed=7).fill().upload()
    c.check(any_stream, 16, c.rng.standard_normal((2, 4, 64)), scale)


@pytest.mark.parametrize("bits", [16, 32])
def test_a_query_that_is_no_number_stays_in_its_row(px_gpu, any_stream, bits):
    c = Call(px_gpu, 1, 128, 32, [300], max_q=6, seed=8).fill().upload()
    q = c.rng.standard_normal((6, 4, 128)).astype(_t(bits))
    clean = c.attend(any_stream, bits, q)
    q[1, 2, 7], q[4, 0, 100] = np.nan, np.inf
    got = c.attend(any_stream, bits, q)
    touched = np.zeros((6, 4), bool)
    touched[1, 2] = touched[4, 0] = True
    assert np.isnan(got[touched]).all() and np.array_equal(got[~touched], clean[~touched])


def test_a_shared_page_and_a_repeated_one(px_gpu, any_stream):
    # two sequences over the same pages, and one page twice in a table
    c = Call(px_gpu, 2, 64, 32, [100, 100, 64], seed=9).fill()
    c.table[1] = c.table[0]
    c.table[2, 1] = c.table[2, 0]
    c.upload()
    c.check(any_stream, 16, c.rng.standard_normal((3, 8, 64)))


def test_long_sequences_split_and_whole(px_gpu, stream):
    px = px_gpu
    rng = np.random.default_rng(10)
    heads, D, P, R = 2, 128, 64, 4
    lens = [9000, 1, 5003]
    c = Call(px, heads, D, P, lens, seed=10)
    p = c.pool  # filled by the whole array: NaN only past the lengths
    p.data[:, :, :P * D] = rng.integers(0, 256, (p.pages, heads, P * D))
    par = np.empty((p.pages, heads, 2, P, 2), np.float16)
    par[..., 0] = rng.uniform(0.02, 0.2, par.shape[:-1])
    par[..., 1] = rng.uniform(-1.5, -0.5, par.shape[:-1])
    p.data[:, :, P * D:] = par.reshape(p.pages, heads, -1).view(np.uint8)
    c.upload()
    q = rng.standard_normal((3, heads * R, D))
    bare = px.Stream()
    for s in (stream, bare):
        for bits in (16, 32):
            c.check(s, bits, q, D ** -0.5)
    bare.destroy()


def test_pool_past_4_gib(px_gpu, stream):
    px = px_gpu
    heads, D, P = 16, 128, 256
    size = px.kv4_page_bytes(heads, D, P)
    pages = (5 << 30) // size
    c = Call(px, heads, D, P, [300], seed=11)
    far = np.array([[pages - 1, pages - 3]], np.int32)
    small = Call(px, heads, D, P, [300], seed=11)
    small.table[:] = [[1, 0]]
    small.fill()
    big = px.DeviceBuffer(pages * size)
    for page, at in ((far[0, 0], 1), (far[0, 1], 0)):
        part = np.ascontiguousarray(small.pool.data[at])
        px.check(px.lib().phx_memcpy_h2d(big.ptr + int(page) * size, part.ctypes.data, size))
    small.upload()
    c.table = far
    c.upload()
    c.cache.pool, c.cache.pages = big.ptr, int(pages)
    q = c.rng.standard_normal((1, 32, D)).astype(np.float16)
    a, b = (x.attend(stream, 16, q) for x in (c, small))
    assert np.array_equal(a, b) and np.abs(a).max() > 0
    # append and read there as well
    k = c.rng.standard_normal((1, heads, D)).astype(np.float16)
    dk, dv, bk, bv = (px.DeviceBuffer.from_array(k) for _ in range(4))
    px.launch_kv4_append(stream, c.cache, c.batch, px.F16, dk, dv)
    px.launch_kv4_read(stream, c.cache, c.batch, px.F16, bk, bv)
    stream.synchronize()
    want = [_stored(k[0, h], np.float16) for h in range(heads)]
    assert np.array_equal(bk.download(np.float16, k.shape)[0], want)
    assert np.array_equal(bv.download(np.float16, k.shape)[0], want)


def _stored(x, t):
    codes, s, m = quantise(x)
    return (codes.astype(np.float32) * np.float32(s) + np.float32(m)).astype(t)


def test_split_plan_and_workspace(px_gpu):
    # what the plan says suffices is used, nothing past it is touched, and with
    # less the launch still is right
    px = px_gpu
    c = Call(px, 1, 64, 32, [4000], seed=12)
    p = c.pool
    p.data[:] = c.rng.integers(0, 256, p.data.shape)
    par = np.empty((p.pages, 1, 2, 32, 2), np.float16)
    par[..., 0], par[..., 1] = 0.1, -0.7
    p.data[:, :, 32 * 64:] = par.reshape(p.pages, 1, -1).view(np.uint8)
    c.upload()
    splits, size = px.kv4_split_plan(c.cache, c.batch, 2)
    assert splits >= 1 and (size > 0) == (splits > 1)
    q = c.rng.standard_normal((1, 2, 64))
    s = px.Stream()
    room = px.DeviceBuffer(size + 4096)
    for cap in {size, max(size // 2, 256), 256, size + 4096 - 256}:
        px.check(px.lib().phx_memset_async(room.ptr, 0xAB, room.nbytes, s.handle))
        px.set_workspace(s, room.ptr, cap)
        c.check(s, 16, q)
        s.synchronize()
        got = room.download(np.uint8, room.nbytes)
        used = min(size, cap)
        assert (got[used:] == 0xAB).all(), "stored past the workspace"
    px.set_workspace(s, 0, 0)
    s.destroy()


@pytest.mark.parametrize("max_q", [1, 40])
def test_captured_and_replayed(px_gpu, max_q):
    px = px_gpu
    heads, Hq, D = 2, 4, 64
    c = Call(px, heads, D, 32, [1500, 40, 900], max_q=max_q, seed=13)
    p = c.pool
    p.data[:] = c.rng.integers(0, 256, p.data.shape)
    par = np.empty((p.pages, heads, 2, 32, 2), np.float16)
    par[..., 0], par[..., 1] = 0.1, -0.7
    p.data[:, :, 32 * 64:] = par.reshape(p.pages, heads, -1).view(np.uint8)
    c.upload()
    s = px.Stream()
    px.bind_workspace(s, 32 << 20)
    shape, kshape = (c.rows, Hq, D), (c.rows, heads, D)
    dq, do, eager = (px.DeviceBuffer(2 * np.prod(shape)) for _ in range(3))
    dk, bk, bv = (px.DeviceBuffer(2 * np.prod(kshape)) for _ in range(3))

    def step(to):
        px.launch_kv4_append(s, c.cache, c.batch, px.F16, dk, dk)
        px.launch_kv4_read(s, c.cache, c.batch, px.F16, bk, bv)
        px.launch_kv4_attention(s, c.cache, c.batch, px.F16, dq, to, Hq, 0.125, True)

    g = Graph(s, lambda: step(do))
    for i in range(4):
        dq.upload(c.rng.standard_normal(shape).astype(np.float16))
        dk.upload(c.rng.standard_normal(kshape).astype(np.float16))
        c.lens -= 5  # a replay reads the lengths of its time
        c.d[1].upload(c.lens)
        do.zero(s)
        g.replay()
        s.synchronize()
        got = do.download(np.uint16, shape)
        step(eager)
        s.synchronize()
        assert np.array_equal(got, eager.download(np.uint16, shape)) and got.any()
    g.destroy()
    px.bind_workspace(s, 0)
    s.destroy()


_FIRST = """
import sys
sys.path[:0] = [{root!r} + "/phobos-lang_amd", {root!r} + "/tests"]
import numpy as np, phobos_amd as px
from hip_graph import Graph
px.init(0)
s = px.Stream()
a = px.DeviceBuffer.from_array(np.ones(128, np.float16))
codes = px.DeviceBuffer.from_array(np.full((128, 16), 9, np.uint8))
w, scales = px.DeviceBuffer(1024), px.DeviceBuffer.from_array(np.ones(16, np.float16))
c = px.DeviceBuffer(32)
c.zero(s)
s.synchronize()

def body():
    px.w4_pack(s, codes, w, 16, 128)
    px.launch_gemv_w4(s, px.F16, a, w, scales, 0, c, 1, 16, 128, 128)

g = Graph(s, body)
assert not c.download(np.uint16, 16).any()  # captured, not run
for _ in range(3):
    c.zero(s)
    g.replay()
    s.synchronize()
    assert (c.download(np.float16, 16) == 128).all()
print("captured first")
"""


def test_a_first_use_may_be_captured():
    # nothing of the library has run: the capture loads the code objects
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", _FIRST.format(root=root)], capture_output=True,
                         text=True, timeout=100)
    assert out.stdout.strip() == "captured first", out.stderr[-2000:]


def test_threads_on_streams_of_their_own(px_gpu):
    import threading
    px = px_gpu
    calls = [Call(px, 2, 64, 32, [300 + 50 * i, 77], seed=20 + i).fill().upload() for i in range(3)]
    qs = [c.rng.standard_normal((2, 8, 64)).astype(np.float16) for c in calls]
    want = []
    for c, q in zip(calls, qs):
        s = px.Stream()
        want.append(c.attend(s, 16, q))
        s.destroy()
    wrong = []

    def work(i):
        s = px.Stream()
        for _ in range(10):
            if not np.array_equal(calls[i].attend(s, 16, qs[i]), want[i]):
                wrong.append(i)
        s.destroy()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_threads_on_one_stream(px_gpu):
    # split launches, whose parts share the stream's workspace
    import threading
    px = px_gpu
    s = px.Stream()
    px.bind_workspace(s, 8 << 20)
    calls = [Call(px, 1, 64, 64, [6000 + 64 * i], seed=50 + i, spare=2) for i in range(3)]
    work = []
    for c in calls:
        c.pool.data[:] = c.rng.integers(0, 256, c.pool.data.shape)
        par = np.empty((c.pool.pages, 1, 2, 64, 2), np.float16)
        par[..., 0], par[..., 1] = 0.1, -0.7
        c.pool.data[:, :, 64 * 64:] = par.reshape(c.pool.pages, 1, -1).view(np.uint8)
        c.upload()
        assert px.kv4_split_plan(c.cache, c.batch, 4)[0] > 1
        q = px.DeviceBuffer.from_array(c.rng.standard_normal((1, 4, 64)).astype(np.float16))
        outs = [px.DeviceBuffer(2 * 4 * 64) for _ in range(20)]
        work.append([lambda o, c=c, q=q: px.launch_kv4_attention(
            s, c.cache, c.batch, px.F16, q, o, 4, 0.125), outs])
    rng = np.random.default_rng(1)
    M, N, K = 40, 1500, 8192
    w = px.DeviceBuffer.from_array(rng.integers(0, 256, px.w4_packed_bytes(N, K)).astype(np.uint8))
    sc = px.DeviceBuffer.from_array((rng.random((256, N)) * 0.01).astype(np.float16))
    a = px.DeviceBuffer.from_array(rng.standard_normal((M, K)).astype(np.float16))
    work.append([lambda o: px.launch_gemv_w4(s, px.F16, a, w, sc, 0, o, M, N, K, 32),
                 [px.DeviceBuffer(2 * M * N) for _ in range(20)]])
    want = []
    for f, outs in work:
        f(outs[0])
        s.synchronize()
        want.append(outs[0].download(np.uint16, outs[0].nbytes // 2).copy())
    threads = [threading.Thread(target=lambda f=f, outs=outs: [f(o) for o in outs])
               for f, outs in work]
    [t.start() for t in threads]
    [t.join() for t in threads]
    s.synchronize()
    for (f, outs), x in zip(work, want):
        for o in outs:
            assert np.array_equal(o.download(np.uint16, o.nbytes // 2), x)
    px.bind_workspace(s, 0)
    s.destroy()


# Enough columns and sequences for whole workgroups of columns
@pytest.mark.parametrize("bits", [16, 32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("size", [1.0, 40.0])
@pytest.mark.parametrize("D,heads,R,P,max_q", [(128, 4, 6, 32, 13), (64, 2, 33, 64, 4),
                                               (128, 4, 70, 64, 1), (64, 4, 1, 32, 65)])
def test_many_columns(px_gpu, stream, bits, causal, size, D, heads, R, P, max_q):
    rng = np.random.default_rng(max_q)
    lens = [2200, 0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257] + list(rng.integers(1, 200, 26))
    counts = rng.integers(0, 4 if max_q > 3 else max_q + 1, 40)
    counts[[0, 9]] = max_q
    counts[2] = min(max_q, 3)  # rows before the first key, in a causal call
    starts = np.concatenate([[0], counts.cumsum()])
    c = Call(px_gpu, heads, D, P, lens, starts, max_q, seed=max_q)
    c.table[20, 0], c.table[21, 1:], c.table[22, :] = -1, c.pool.pages, -5
    c.table[0, 3], c.table[0, 40 // (P // 32)] = 1 << 30, -1
    c.fill().upload()
    q = c.rng.standard_normal((c.rows, heads * R, D)) * size
    q[-1] = 0
    q[-2, 0] *= 2.0 ** -16
    got = c.check(stream, bits, q, D ** -0.5, causal, pad=8, extra=2)
    # a row that is no number stays in its row
    q[-3, 1, 5] = np.inf
    again = c.attend(stream, bits, q.astype(_t(bits)), D ** -0.5, causal)
    assert not np.isfinite(again[-3, 1]).any() or c.lens[np.searchsorted(starts, len(q) - 3, "right") - 1] < 1
    again[-3, 1] = got[-3, 1]
    assert np.array_equal(again, got.astype(_t(bits)))
