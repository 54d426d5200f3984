"""phx_pages_copy and phx_pages_apply: bytes moved, bytes left alone."""
import numpy as np
import pytest

from hip_graph import Graph

pytestmark = pytest.mark.gpu


def _pool(px, layers, pages, words, stride_words, seed):
    host = np.random.default_rng(seed).integers(0, 1 << 32, layers * stride_words + 4,
                                                dtype=np.uint32)
    return host, px.DeviceBuffer.from_array(host)


@pytest.mark.parametrize("layers,pages,words,pad,copies", [
    (1, 2, 4, 0, 1), (3, 7, 20, 8, 3), (2, 40, 4 * 1024, 0, 20), (1, 5, 4 * 1024 + 4, 4, 2),
    (5, 1500, 12, 16, 700), (1, 1000, 8, 0, 449)])
def test_copies(px_gpu, stream, layers, pages, words, pad, copies):
    px = px_gpu
    stride = pages * words + pad
    host, buf = _pool(px, layers, pages, words, stride, pages)
    rng = np.random.default_rng(words)
    order = rng.permutation(pages)
    dst = order[:copies]
    src = rng.choice(order[copies:], copies)  # some several times
    px.pages_copy(stream, buf, pages, 4 * words, src, dst, layers, 4 * stride)
    want = host.copy()
    for layer in range(layers):
        part = want[layer * stride:layer * stride + pages * words].reshape(pages, words)
        part[dst] = part[src]
    stream.synchronize()
    assert np.array_equal(buf.download(np.uint32, host.shape), want)


def test_copies_of_a_page_to_itself_and_none(px_gpu, stream):
    px = px_gpu
    host, buf = _pool(px, 1, 4, 16, 64, 1)
    px.pages_copy(stream, buf, 4, 64, [1, 0], [1, 2])
    px.pages_copy(stream, buf, 4, 64, [], [])
    px.pages_copy(stream, buf, 4, 64, [0], [1], 0, 0)
    host[32:48] = host[0:16]
    stream.synchronize()
    assert np.array_equal(buf.download(np.uint32, host.shape), host)


def test_addresses_past_32_bits(px_gpu, stream):
    px = px_gpu
    page, pages = 1 << 26, 80  # 5 GiB
    buf = px.DeviceBuffer(page * pages)
    mark = np.arange(page // 4, dtype=np.uint32)
    px.check(px.lib().phx_memcpy_h2d(buf.ptr + 70 * page, mark.ctypes.data, page))
    px.pages_copy(stream, buf, pages, page, [70], [79])
    stream.synchronize()
    got = np.empty_like(mark)
    px.check(px.lib().phx_memcpy_d2h(got.ctypes.data, buf.ptr + 79 * page, page))
    assert np.array_equal(got, mark)
    buf.free()


def test_apply_runs_forks_and_compactions(px_gpu, stream):
    px = px_gpu
    pages, P, layers, words = 12, 4, 3, 8
    host, buf = _pool(px, layers, pages, words, pages * words, 9)
    pool = px.Pages(pages, P)
    view = host[:layers * pages * words].reshape(layers, pages, words)
    a, b = pool.new(), pool.new()
    pool.resize(a, 10)
    pool.resize(b, 3)
    c = pool.fork(a)
    pool.resize(c, 11)
    kept = view[:, pool.table(a)].copy()
    pool.apply(stream, buf, 4 * words, layers, 4 * pages * words)
    assert pool.stats() == (5, 5, 0)
    pool.free(a)
    pool.free(b)
    pool.compact()
    pool.apply(stream, buf, 4 * words, layers, 4 * pages * words)
    assert pool.stats() == (3, 3, 0)
    stream.synchronize()
    got = buf.download(np.uint32, host.shape)[:view.size].reshape(view.shape)
    assert np.array_equal(got[:, pool.table(c)], kept)


def test_copies_in_a_captured_graph(px_gpu):
    px = px_gpu
    host = np.arange(6 * 64, dtype=np.uint32).reshape(6, 64)
    buf, s = px.DeviceBuffer.from_array(host), px.Stream()
    g = Graph(s, lambda: px.pages_copy(s, buf, 6, 256, [0, 0], [3, 5]))
    for i in range(4):
        host[0] = 1000 + i
        buf.upload(host[:1])
        g.replay()
        s.synchronize()
        got = buf.download(np.uint32, host.shape)
        assert (got[[0, 3, 5]] == 1000 + i).all() and np.array_equal(got[[1, 2, 4]], host[[1, 2, 4]])
    g.destroy()
    s.destroy()


def test_apply_is_no_part_of_a_graph(px_gpu):
    # replayed, it would copy the old pages over what was written since
    px = px_gpu
    host = np.arange(6 * 64, dtype=np.uint32).reshape(6, 64)
    buf, s = px.DeviceBuffer.from_array(host), px.Stream()
    pool = px.Pages(6, 4)
    a = pool.new()
    pool.resize(a, 2)
    b = pool.fork(a)
    pool.resize(b, 3)
    refused = []

    def body():
        px.pages_copy(s, buf, 6, 256, [3], [4])
        try:
            pool.apply(s, buf, 256)
        except px.PhxError as e:
            refused.append(e.code)

    g = Graph(s, body)
    assert refused == [px.PHX_E_INVALID] and pool.stats()[2] == 1
    pool.apply(s, buf, 256)
    assert pool.stats()[2] == 0
    g.replay()
    # with nothing pending there is nothing to launch, captured or not
    quiet = Graph(s, lambda: (pool.apply(s, buf, 256), px.pages_copy(s, buf, 6, 256, [3], [5])))
    quiet.replay()
    s.synchronize()
    got = buf.download(np.uint32, host.shape)
    assert np.array_equal(got[pool.table(b)[0]], host[0])
    assert np.array_equal(got[[4, 5]], host[[3, 3]])
    g.destroy()
    quiet.destroy()
    s.destroy()
