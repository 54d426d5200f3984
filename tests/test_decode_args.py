"""What the decode operators refuse, before any device is touched: without one
a good call ends in PHX_E_NOT_INIT and a bad one in PHX_E_INVALID."""
import ctypes
import subprocess
import sys

import numpy as np
import pytest

import phobos_amd as px

A = 1 << 20  # an address that passes the checks; nothing is launched


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


def _gemv(**kw):
    a = dict(dtype=px.F16, a=A, w=A, scales=A, zeros=0, c=A, M=1, N=5, K=40, group=32, alpha=1.0,
             beta=0.0, lda=0, ldc=0)
    a.update(kw)
    return _rc(lambda: px.launch_gemv_w4(None, a.pop("dtype"), *a.values()))


@pytest.mark.parametrize("ok", [{}, {"M": 64}, {"M": 0, "a": 0, "c": 0}, {"K": 8}, {"group": 64},
                                {"group": 128}, {"lda": 48, "ldc": 7}, {"N": (1 << 25) - 1}, {"dtype": px.F32, "lda": 44},
                                {"scales": A + 2, "zeros": A + 1, "c": A + 2}])
def test_gemv_takes(ok):
    assert _gemv(**ok) == px.PHX_E_NOT_INIT


@pytest.mark.parametrize("bad", [
    {"dtype": 2}, {"dtype": -1}, {"M": -1}, {"M": 65}, {"N": 0}, {"N": -5}, {"K": 0}, {"K": 4},
    {"K": 44}, {"K": -8}, {"N": 1 << 31}, {"N": 1 << 25}, {"K": 1 << 31}, {"group": 0}, {"group": 16}, {"group": -32},
    {"group": 256}, {"lda": 32}, {"lda": 44}, {"ldc": 4}, {"lda": -40}, {"dtype": px.F32, "lda": 42},
    {"lda": 1 << 40}, {"lda": 1 << 62}, {"ldc": 1 << 62}, {"a": 0}, {"w": 0}, {"scales": 0}, {"c": 0},
    {"a": A + 8}, {"w": A + 4}, {"scales": A + 1}, {"c": A + 1}, {"dtype": px.F32, "c": A + 2}])
def test_gemv_refuses(bad):
    assert _gemv(**bad) == px.PHX_E_INVALID
    assert "gemv_w4" in px.lib().phx_last_error().decode()


def test_w4_pack():
    assert px.w4_packed_bytes(16, 128) == 1024 and px.w4_packed_bytes(17, 129) == 4096
    assert px.w4_packed_bytes(-1, 128) == 0 and px.w4_packed_bytes(0, 128) == 0
    pack = lambda *a: _rc(lambda: px.w4_pack(None, *a))  # noqa: E731
    assert pack(A, A, 5, 7) == pack(0, 0, 0, 7) == px.PHX_E_NOT_INIT
    for bad in [(0, A, 5, 7), (A, 0, 5, 7), (A, A + 8, 5, 7), (A, A, -1, 7), (A, A, 5, 1 << 31)]:
        assert pack(*bad) == px.PHX_E_INVALID


def _kv4(op, cache=None, batch=None, **kw):
    c = dict(pool=A, pages=9, heads=2, head_dim=64, page_tokens=32)
    b = dict(table=A, table_stride=3, lens=A, q_starts=0, batch=2, max_q=1, max_len=96, rows=2)
    c.update(cache or {})
    b.update(batch or {})
    a = dict(dtype=px.F16, x=A, y=A, q_heads=4, ldx=0, ldy=0)
    a.update(kw)
    c, b = px.Kv4Cache(*c.values()), px.Kv4Batch(*b.values())
    if op == "attend":
        return _rc(lambda: px.launch_kv4_attention(None, c, b, a["dtype"], a["x"], a["y"],
                                                   a["q_heads"], 0.125, True, a["ldx"], a["ldy"]))
    f = px.launch_kv4_append if op == "append" else px.launch_kv4_read
    return _rc(lambda: f(None, c, b, a["dtype"], a["x"], a["y"], a["ldx"], a["ldy"]))


OPS = ["append", "read", "attend"]


@pytest.mark.parametrize("op", OPS)
def test_kv4_takes(op):
    none = dict(x=0, y=0)
    assert _kv4(op) == px.PHX_E_NOT_INIT
    assert _kv4(op, dict(head_dim=128, page_tokens=256)) == px.PHX_E_NOT_INIT
    assert _kv4(op, batch=dict(q_starts=A, max_q=7, rows=5)) == px.PHX_E_NOT_INIT
    assert _kv4(op, batch=dict(table=0, table_stride=0)) == px.PHX_E_NOT_INIT
    for empty in (dict(batch=0), dict(max_q=0), dict(rows=0)):
        assert _kv4(op, batch=dict(empty, lens=0, table=0), **none) == px.PHX_E_NOT_INIT
    assert _kv4(op, ldx=264, ldy=512) == px.PHX_E_NOT_INIT
    assert _kv4(op, dtype=px.F32, ldx=260) == px.PHX_E_NOT_INIT


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("what,bad", [("cache", x) for x in (
    dict(pool=0), dict(pool=A + 16), dict(pages=0), dict(pages=-1), dict(pages=1 << 31),
    dict(heads=0), dict(heads=-2), dict(heads=1025), dict(head_dim=0), dict(head_dim=96),
    dict(head_dim=256), dict(page_tokens=0), dict(page_tokens=16), dict(page_tokens=48),
    dict(page_tokens=512))] + [("batch", x) for x in (
        dict(batch=-1), dict(batch=65536), dict(max_q=-1), dict(max_q=1 << 31), dict(rows=-1),
        dict(rows=1 << 31), dict(table_stride=-1), dict(table_stride=1 << 31), dict(max_len=-1),
        dict(max_len=1 << 31), dict(lens=0), dict(lens=A + 2), dict(table=0), dict(table=A + 1),
        dict(q_starts=A + 2))] + [("args", x) for x in (
            dict(dtype=2), dict(x=0), dict(y=0), dict(x=A + 8), dict(y=A + 4), dict(ldx=127),
            dict(ldx=300), dict(ldy=-256), dict(ldy=1 << 50), dict(dtype=px.F32, ldx=258))])
def test_kv4_refuses(op, what, bad):
    kw = dict(bad) if what == "args" else {what: bad}
    assert _kv4(op, **kw) == px.PHX_E_INVALID
    assert "kv4_" in px.lib().phx_last_error().decode()


@pytest.mark.parametrize("op", OPS)
def test_more_rows_than_a_launch_takes(op):
    # with q_starts max_q is a bound that no tensor has to hold
    few = dict(q_starts=A, batch=100, rows=3)
    assert _kv4(op, batch=dict(few, max_q=1000)) == px.PHX_E_NOT_INIT
    assert _kv4(op, batch=dict(few, batch=65535, max_q=(1 << 31) - 1)) == px.PHX_E_INVALID
    assert "too many" in px.lib().phx_last_error().decode()


def test_kv4_attention_heads():
    for heads in (0, -2, 3, 1 << 20):
        assert _kv4("attend", q_heads=heads) == px.PHX_E_INVALID
    assert _kv4("attend", q_heads=2) == _kv4("attend", q_heads=32) == px.PHX_E_NOT_INIT


@pytest.mark.parametrize("f", ["append", "read", "attention"])
def test_kv4_null_descriptors(f):
    L = px.lib()
    c, b = px.Kv4Cache(A, 9, 2, 64, 32), px.Kv4Batch(A, 3, A, 0, 2, 1, 96, 2)
    more = [4, 0.125, 1, 0, 0] if f == "attention" else [0, 0]
    for cache, batch in ((None, b), (c, None)):
        assert getattr(L, "phx_kv4_" + f)(None, cache, batch, 1, A, A, *more) == px.PHX_E_INVALID
    assert L.phx_kv4_split_plan(None, b, 4, None, None) == px.PHX_E_INVALID
    assert L.phx_kv4_split_plan(c, None, 4, None, None) == px.PHX_E_INVALID
    assert L.phx_kv4_split_plan(c, b, 3, None, None) == px.PHX_E_INVALID
    assert L.phx_kv4_split_plan(c, b, 4, None, None) == 0


def test_page_bytes():
    assert px.kv4_page_bytes(1, 64, 32) == 32 * 72
    assert px.kv4_page_bytes(8, 128, 64) == 8 * 64 * 136
    for bad in [(0, 64, 32), (1, 80, 32), (1, 64, 33), (-1, 64, 32)]:
        assert px.kv4_page_bytes(*bad) == 0


def _copy(src, dst, pool=A, pages=8, page_bytes=4096, layers=2, stride=8 * 4096):
    return _rc(lambda: px.pages_copy(None, pool, pages, page_bytes, src, dst, layers, stride))


def test_pages_copy():
    for ok in [([0, 0, 1], [2, 3, 4]), ([], []), ([5], [5]), ([7, 5], [0, 5])]:
        assert _copy(*ok) == px.PHX_E_NOT_INIT
    assert _copy([0], [1], layers=0, pool=0) == px.PHX_E_NOT_INIT
    assert _copy([0], [1], layers=1, stride=0) == px.PHX_E_NOT_INIT
    for bad in [([0, 1], [2, 2]), ([0, 1], [1, 2]), ([-1], [0]), ([0], [-1]),
                ([8], [0]), ([0], [8])]:
        assert _copy(*bad) == px.PHX_E_INVALID, bad
    for kw in [dict(pool=0), dict(pool=A + 8), dict(pages=0), dict(page_bytes=0),
               dict(page_bytes=24), dict(layers=-1), dict(layers=65536), dict(stride=4096),
               dict(stride=8 * 4096 + 8), dict(stride=0)]:
        assert _copy([0], [1], **kw) == px.PHX_E_INVALID, kw
    assert px.lib().phx_pages_copy(None, A, 8, 4096, None, None, 1, 1, 0) == px.PHX_E_INVALID
    assert _rc(lambda: px.pages_copy(None, A, 8, 4096, [0, 1], [2])) == px.PHX_E_INVALID


def test_page_lists():
    # numbers that would wrap around to a page, arrays of every kind
    for bad in ([1 << 32], np.array([1 << 32]), np.array([(1 << 32) + 1], np.uint64), [-(1 << 40)],
                [[0]], 0, np.int64(0)):
        assert _copy(bad, [1]) == px.PHX_E_INVALID, bad
        assert _copy([1], bad) == px.PHX_E_INVALID, bad
    held = np.array([0, 3], np.int32)
    held.flags.writeable = False
    for ok in (held, held.astype(np.int64), (0, 3), np.array([0, 9, 3, 9])[::2], held.astype(np.uint8)):
        assert _copy(ok, [1, 2]) == px.PHX_E_NOT_INIT


def test_a_copy_onto_a_kept_page_is_still_one_destination():
    # 2 -> 2 is left out, and then 2 is the destination of one copy only
    assert _copy([2, 0], [2, 2]) == px.PHX_E_NOT_INIT


def test_pages_apply_keeps_what_it_could_not_launch():
    pool = px.Pages(8, 4)
    a = pool.new()
    pool.resize(a, 2)
    pool.resize(pool.fork(a), 3)
    for _ in range(2):
        with pytest.raises(px.PhxError):
            pool.apply(None, A, 4096)
        assert pool.stats()[2] == 1


def test_buffers_are_measured():
    # a DeviceBuffer smaller than the call reaches is refused on the host
    buf = px.DeviceBuffer.__new__(px.DeviceBuffer)
    buf.ptr, buf.nbytes = A, 100
    assert _gemv(a=buf, K=40, M=2) == px.PHX_E_INVALID  # needs 160 B
    assert _gemv(w=buf) == _gemv(scales=buf, N=40) == _gemv(c=buf, M=11) == px.PHX_E_INVALID
    assert _gemv(a=buf, K=40, M=1) == px.PHX_E_NOT_INIT
    assert _kv4("append", x=buf) == _kv4("attend", y=buf) == px.PHX_E_INVALID
    buf.ptr = 0  # nothing of it is freed


def test_w4_quantize():
    rng = np.random.default_rng(4)
    b = rng.standard_normal((70, 9))
    b[:32, 3] = 0
    b[:, 5] = np.abs(b[:, 5])
    for group in (32, 64, 128):
        codes, scales, zeros = px.w4_quantize(b, group)
        g = np.arange(70) // group
        back = (codes.astype(np.float64) - zeros[g]) * scales.astype(np.float64)[g]
        # half a step, and what the f16 scale and the whole zero point shift the range by
        assert (np.abs(back - b) <= scales.astype(np.float64)[g] * (1.0 + 15 * 2.0 ** -11)).all()
        assert (back[:32, 3] == 0).all() or group > 32
        assert codes.max() <= 15 and zeros.max() <= 15


def test_an_uninitialised_process_is_refused():
    # the module's fixture holds; a child process makes sure of it
    code = ("import sys; sys.path[:0] = [%r]; import phobos_amd as px\n"
            "try: px.launch_gemv_w4(None, px.F16, 16, 16, 16, 0, 16, 1, 1, 8, 32)\n"
            "except px.PhxError as e: print(e.code)" % px.ROOT)
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert out.stdout.strip() == str(px.PHX_E_NOT_INIT), out.stderr
    assert ctypes.sizeof(px.Kv4Cache) == 32 and ctypes.sizeof(px.Kv4Batch) == 64


def test_pages_apply_measures_its_pool():
    # every page of every layer has to lie in the buffer, whichever are copied
    pool = px.Pages(8, 4)
    a = pool.new()
    pool.resize(a, 2)
    pool.resize(pool.fork(a), 3)
    buf = px.DeviceBuffer.__new__(px.DeviceBuffer)
    buf.ptr = A
    for nbytes, layers, stride, rc in [(8 * 64, 1, 0, px.PHX_E_NOT_INIT), (8 * 64 - 1, 1, 0, px.PHX_E_INVALID),
                                       (9 * 64 + 8 * 64, 2, 9 * 64, px.PHX_E_NOT_INIT),
                                       (9 * 64 + 8 * 64 - 1, 2, 9 * 64, px.PHX_E_INVALID)]:
        buf.nbytes = nbytes
        assert _rc(lambda: pool.apply(None, buf, 64, layers, stride)) == rc, (nbytes, layers)
        assert pool.stats()[2] == 1
    buf.ptr = 0  # nothing of it is freed


def test_layers_that_wrap_around():
    # (a negative distance arrives as one of nearly 2^64 bytes)
    buf = px.DeviceBuffer.__new__(px.DeviceBuffer)
    buf.ptr, buf.nbytes = 1 << 40, 16 * 4096
    for pool in (1 << 40, buf):
        for layers, stride in [(2, -8 * 4096), (2, (1 << 64) - 8 * 4096), (3, 1 << 63), (65535, 1 << 49),
                               (2, -(1 << 30)), (5, -(1 << 62))]:
            assert _copy([0], [1], pool=pool, layers=layers, stride=stride) == px.PHX_E_INVALID, stride
    assert _copy([0], [1], pool=(1 << 64) - 16 * 4096, layers=2) == px.PHX_E_INVALID
    assert _copy([0], [1], pool=(1 << 64) - 17 * 4096, layers=2) == px.PHX_E_NOT_INIT
    assert _copy([0], [1], pool=(1 << 64) - 8 * 4096, layers=1) == px.PHX_E_INVALID
    buf.ptr = 0  # nothing of it is freed


def test_page_numbers_are_whole():
    nan = float("nan")
    for bad in ([1.7], [1.0], np.array([0.7]), np.array([3.0], np.float32), [nan], ["1"], [None], [True],
                np.array([True]), [1 + 0j], [1 << 70], [-(1 << 63) - 1], [(1 << 31)], [-(1 << 31) - 1],
                None, "1", [[1], [2, 3]]):
        assert _copy(bad, [1]) == px.PHX_E_INVALID, bad
        assert _copy([0], bad) == px.PHX_E_INVALID, bad
    for ok in (np.array([0], t) for t in (np.int8, np.uint16, np.uint32, np.uint64, ">i4", ">i8")):
        assert _copy(ok, [1]) == px.PHX_E_NOT_INIT, ok.dtype
    torch = pytest.importorskip("torch")
    for ok in (torch.tensor([0, 3]), torch.tensor([0, 3], dtype=torch.int32), torch.arange(4)[::3]):
        assert _copy(ok, [1, 2]) == px.PHX_E_NOT_INIT
    for bad in (torch.tensor([0.5]), torch.tensor([True]), torch.tensor(0), torch.tensor([1 << 32])):
        assert _copy(bad, [1]) == px.PHX_E_INVALID
    for none in (np.int64(0), torch.tensor(0), 0):
        assert _copy(none, []) == px.PHX_E_INVALID
    # an empty list has no kind
    assert _copy([], np.empty(0)) == _copy((), torch.empty(0)) == px.PHX_E_NOT_INIT


def test_pages_apply_of_no_layers_keeps_its_copies():
    pool = px.Pages(8, 4)
    a = pool.new()
    pool.resize(a, 2)
    pool.resize(pool.fork(a), 3)
    for layers in (0, -1, 65536):
        assert _rc(lambda: pool.apply(None, A, 4096, layers, 8 * 4096)) == px.PHX_E_INVALID
        assert pool.stats()[2] == 1


def test_sizes_that_would_wrap_around():
    for far in (1 << 32, 1 << 31, -(1 << 32), 1 << 64):
        assert _rc(lambda: px.Pages(8 + far, 4)) == px.PHX_E_INVALID
        assert _rc(lambda: px.Pages(8, 4 + far)) == px.PHX_E_INVALID
        for i in range(3):
            sizes = [2, 64, 32]
            sizes[i] += far
            assert _rc(lambda: px.Kv4Cache(A, 9, *sizes)) == px.PHX_E_INVALID
            assert px.kv4_page_bytes(*sizes) == 0
    assert _rc(lambda: px.Kv4Cache(A, 9, 2, head_dim=64 + (1 << 32), page_tokens=32)) == px.PHX_E_INVALID
    c = px.Kv4Cache(A, 9, 2, head_dim=64, page_tokens=32)
    assert (c.pool, c.pages, c.heads, c.head_dim, c.page_tokens) == (A, 9, 2, 64, 32)
    assert px.Kv4Cache().heads == 0


def test_w4_quantize_refuses_what_no_scale_holds():
    b = np.zeros((64, 3))
    b[40, 1] = 15 * 65504.0
    codes, scales, zeros = px.w4_quantize(b, 32)
    assert scales[1, 1] == 65504 and codes[40, 1] == 15
    for bad in (15.1 * 65504 * 1.001, -1e300, np.nan, np.inf, -np.inf):
        b[40, 1] = bad
        assert _rc(lambda: px.w4_quantize(b, 32)) == px.PHX_E_INVALID, bad


def test_w4_quantize_of_tiny_weights():
    # scales below f16's normal numbers are up to half of themselves off when
    # rounded to the nearest, which left the largest weights out of reach
    rng = np.random.default_rng(6)
    for size in 2.0 ** -np.arange(8.0, 24.0):
        b = (rng.random((64, 40)) - 0.3) * size
        codes, scales, zeros = px.w4_quantize(b, 32)
        s = scales.astype(np.float64)[np.arange(64) // 32]
        back = (codes.astype(np.float64) - zeros[np.arange(64) // 32]) * s
        assert (np.abs(back - b) <= s * (1.0 + 15 * 2.0 ** -11)).all(), size
        # no step is wider than the range takes, but for the f16 it is rounded to
        want = np.stack([np.ptp(np.concatenate([b[g:g + 32], b[:1] * 0]), axis=0) for g in (0, 32)]) / 15
        assert (scales <= want * (1 + 2.0 ** -11) + 2.0 ** -24).all(), size
