"""Python host mirror of the phobos leaf-kernel launch interface on MI355X.

This is a thin ctypes layer over libphobos_hip.so (the C ABI in
include/phobos_hip.h).  It mirrors the reference's host-side launch helpers:

  launch_saxpy  -- phobos-bench/src/main.rs:1227-1239 (the saxpy launch! call)
  launch_gemm   -- phobos-bench/src/main.rs:290-327
  launch_flash  -- phobos-bench/src/main.rs:334-371
  compute       -- phobos-pod/src/engine.rs:582-647 (exploded-memref marshalling)

Every call goes to the gfx950 code objects through hipModuleLaunchKernel.
There is no CPU fallback: if the library or a code object is missing, or no
GPU is present, the call raises.
"""
import array
import ctypes
import os
import re

import numpy as np

_PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(_PKG)  # phobos-lang_amd/
LIB_DIR = os.path.join(ROOT, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libphobos_hip.so")
HEADER = os.path.join(os.path.dirname(ROOT), "include", "phobos_hip.h")

# phx_kernel ids (include/phobos_hip.h)
SAXPY_FP32 = 0
GEMM_FP32 = 1
GEMM_FP16TC_FP32ACC = 2
GEMM_FP16 = 3
FLASH_FP32 = 4
FLASH_FP16 = 5
MATMUL = 6
MATMUL_INIT = 7
FLASH_FP32_BH = 8
FLASH_FP16_BH = 9
NUM_KERNELS = 10

KERNEL_NAMES = {
    SAXPY_FP32: "saxpy_fp32", GEMM_FP32: "gemm_fp32",
    GEMM_FP16TC_FP32ACC: "gemm_fp16tc_fp32acc", GEMM_FP16: "gemm_fp16",
    FLASH_FP32: "flash_fp32", FLASH_FP16: "flash_fp16", MATMUL: "matmul",
    MATMUL_INIT: "matmul_init", FLASH_FP32_BH: "flash_fp32_bh", FLASH_FP16_BH: "flash_fp16_bh",
}

CODE_OBJECTS = ["saxpy_fp32.hsaco", "gemm_fp32.hsaco", "gemm_fp16tc_fp32acc.hsaco",
                "gemm_fp16.hsaco", "flash_attention_fp32.hsaco", "flash_attention_fp16.hsaco",
                "matmul_cluster_fp32.hsaco", "gemv_w4.hsaco", "kv4.hsaco",
                "kv4_attend.hsaco", "pages.hsaco", "f8_rows.hsaco", "gemm_f8.hsaco"]

# phx_dtype of the decode and the 8-bit operators
F32 = 0
F16 = 1

PHX_E_INVALID = 1001
PHX_E_NOT_INIT = 1002
PHX_E_NOT_FOUND = 1003
PHX_E_EXHAUSTED = 1004


class PhxError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"phx error {code}: {msg}")
        self.code = code


class TileArg(ctypes.Structure):
    _fields_ = [("addr", ctypes.c_uint64), ("rank", ctypes.c_uint32),
                ("shape", ctypes.c_uint64 * 3)]


class ScalarArg(ctypes.Structure):
    _fields_ = [("pos", ctypes.c_uint32), ("bytes", ctypes.c_uint32), ("bits", ctypes.c_uint64)]


def _fit32(*sizes):
    """Whether none would wrap around as an int32."""
    return all(-(1 << 31) <= x < 1 << 31 for x in sizes)


class Kv4Cache(ctypes.Structure):
    """phx_kv4_cache: a pool of 4-bit key and value pages (device address)."""
    _fields_ = [("pool", ctypes.c_uint64), ("pages", ctypes.c_int64), ("heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("page_tokens", ctypes.c_int32)]

    def __init__(self, pool=0, pages=0, heads=0, head_dim=0, page_tokens=0):
        if not _fit32(heads, head_dim, page_tokens):
            raise PhxError(PHX_E_INVALID, f"cache of {heads} heads of {head_dim}, {page_tokens} tokens a page")
        super().__init__(pool, pages, heads, head_dim, page_tokens)


class Kv4Batch(ctypes.Structure):
    """phx_kv4_batch: the sequences of a call (device addresses of i32 arrays)."""
    _fields_ = [("table", ctypes.c_uint64), ("table_stride", ctypes.c_int64),
                ("lens", ctypes.c_uint64), ("q_starts", ctypes.c_uint64),
                ("batch", ctypes.c_int64), ("max_q", ctypes.c_int64),
                ("max_len", ctypes.c_int64), ("rows", ctypes.c_int64)]


class F8Rows(ctypes.Structure):
    """phx_f8_rows: rows in 8 bits, e4m3 codes and a scale for each 128 (device
    addresses)."""
    _fields_ = [("codes", ctypes.c_uint64), ("scales", ctypes.c_uint64), ("rows", ctypes.c_int64),
                ("k", ctypes.c_int64), ("ld", ctypes.c_int64), ("lds", ctypes.c_int64)]


class F8Weights(ctypes.Structure):
    """phx_f8_weights: weights in 8 bits, e4m3 codes and a scale for each 128 x 128
    (device addresses)."""
    _fields_ = [("codes", ctypes.c_uint64), ("scales", ctypes.c_uint64),
                ("experts", ctypes.c_int64), ("n", ctypes.c_int64), ("k", ctypes.c_int64)]


_LIB = None
_INIT = False

_u64 = ctypes.c_uint64
_i64 = ctypes.c_int64
_vp = ctypes.c_void_p
_sz = ctypes.c_size_t
_u32a3 = ctypes.c_uint32 * 3


def header_symbols():
    """Every phx_* function declared in include/phobos_hip.h."""
    with open(HEADER) as f:
        text = f.read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(phx_[a-z0-9_]+)\s*\(", text)))


def lib():
    """Load libphobos_hip.so (raises if it has not been built)."""
    global _LIB
    if _LIB is not None:
        return _LIB
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} is missing: build the backend first "
                           "(python -c 'import __graft_entry__ as g; g.build()')")
    L = ctypes.CDLL(LIB_PATH)
    L.phx_last_error.restype = ctypes.c_char_p
    L.phx_init.argtypes = [ctypes.c_int, ctypes.c_char_p]
    L.phx_device_info.argtypes = [ctypes.c_char_p, _sz, ctypes.POINTER(ctypes.c_int),
                                  ctypes.POINTER(ctypes.c_int), ctypes.POINTER(_sz),
                                  ctypes.POINTER(ctypes.c_int)]
    L.phx_malloc.argtypes = [ctypes.POINTER(_u64), _sz]
    L.phx_free.argtypes = [_u64]
    L.phx_host_alloc.argtypes = [ctypes.POINTER(_vp), _sz]
    L.phx_host_free.argtypes = [_vp]
    L.phx_memcpy_h2d.argtypes = [_u64, _vp, _sz]
    L.phx_memcpy_d2h.argtypes = [_vp, _u64, _sz]
    L.phx_kernel_by_name.argtypes = [ctypes.POINTER(ctypes.c_int), ctypes.c_char_p, ctypes.c_char_p]
    L.phx_launch_by_name.argtypes = [ctypes.c_char_p, ctypes.c_char_p, _vp, _vp, _vp,
                                     ctypes.POINTER(ctypes.c_void_p)]
    L.phx_memcpy_d2d.argtypes = [_u64, _u64, _sz]
    L.phx_memcpy_h2d_async.argtypes = [_u64, _vp, _sz, _vp]
    L.phx_memcpy_d2h_async.argtypes = [_vp, _u64, _sz, _vp]
    L.phx_memset_async.argtypes = [_u64, ctypes.c_int, _sz, _vp]
    L.phx_stream_create.argtypes = [ctypes.POINTER(_vp)]
    L.phx_stream_destroy.argtypes = [_vp]
    L.phx_stream_synchronize.argtypes = [_vp]
    L.phx_stream_set_workspace.argtypes = [_vp, _u64, _sz]
    L.phx_stream_get_workspace.argtypes = [_vp, ctypes.POINTER(_u64), ctypes.POINTER(_sz)]
    L.phx_event_create.argtypes = [ctypes.POINTER(_vp)]
    L.phx_event_destroy.argtypes = [_vp]
    L.phx_event_record.argtypes = [_vp, _vp]
    L.phx_event_query.argtypes = [_vp]
    L.phx_event_synchronize.argtypes = [_vp]
    L.phx_event_elapsed_ms.argtypes = [ctypes.POINTER(ctypes.c_float), _vp, _vp]
    L.phx_module_load_data.argtypes = [ctypes.POINTER(_vp), ctypes.c_char_p, _sz]
    L.phx_module_load_file.argtypes = [ctypes.POINTER(_vp), ctypes.c_char_p]
    L.phx_module_unload.argtypes = [_vp]
    L.phx_module_get_function.argtypes = [ctypes.POINTER(_vp), _vp, ctypes.c_char_p]
    L.phx_builtin_function.argtypes = [ctypes.POINTER(_vp), ctypes.c_int]
    L.phx_kernel_abi.argtypes = [ctypes.c_int, ctypes.POINTER(ctypes.c_int), _u32a3]
    L.phx_launch.argtypes = [_vp, _u32a3, _u32a3, ctypes.c_uint32, _vp, ctypes.POINTER(_vp)]
    L.phx_grid_for.argtypes = [ctypes.c_int, ctypes.POINTER(_i64), ctypes.c_int, _u32a3, _u32a3]
    L.phx_check_shape.argtypes = [ctypes.c_int, ctypes.POINTER(_i64), ctypes.c_int]
    L.phx_split_plan.argtypes = [ctypes.c_int, ctypes.POINTER(_i64), ctypes.c_int,
                                 ctypes.POINTER(ctypes.c_int), ctypes.POINTER(_sz)]
    L.phx_plan_get.argtypes = [ctypes.c_int, ctypes.POINTER(_i64), ctypes.c_int,
                               ctypes.POINTER(Plan)]
    L.phx_plan_pin.argtypes = [ctypes.c_int, ctypes.POINTER(_i64), ctypes.c_int,
                               ctypes.POINTER(Plan)]
    L.phx_compute.argtypes = [_vp, ctypes.c_int, ctypes.POINTER(TileArg), ctypes.c_uint32,
                              ctypes.POINTER(ScalarArg), ctypes.c_uint32, _u32a3, _u32a3, _vp]
    L.phx_saxpy.argtypes = [_vp, _u64, _u64, _u64, _i64, ctypes.c_float]
    L.phx_gemm.argtypes = [_vp, ctypes.c_int, _u64, _u64, _u64, _i64, _i64, _i64,
                           ctypes.c_float, ctypes.c_float]
    L.phx_matmul_init.argtypes = [_vp, _u64, _i64, _i64, ctypes.c_float]
    L.phx_flash_attention.argtypes = [_vp, ctypes.c_int, _u64, _u64, _u64, _u64, _i64, _i64,
                                      _i64, ctypes.c_float]
    L.phx_flash_attention_bh.argtypes = [_vp, ctypes.c_int, _u64, _u64, _u64, _u64, _i64, _i64,
                                         _i64, _i64, ctypes.c_float]
    L.phx_flash_attention_bh_noalloc.argtypes = L.phx_flash_attention_bh.argtypes
    L.phx_w4_packed_bytes.argtypes = [_i64, _i64]
    L.phx_w4_packed_bytes.restype = _sz
    L.phx_w4_pack.argtypes = [_vp, _u64, _u64, _i64, _i64]
    L.phx_gemv_w4.argtypes = [_vp, ctypes.c_int] + [_u64] * 5 + [_i64] * 4 + \
        [ctypes.c_float] * 2 + [_i64] * 2
    _cache, _batch = ctypes.POINTER(Kv4Cache), ctypes.POINTER(Kv4Batch)
    L.phx_kv4_page_bytes.argtypes = [ctypes.c_int32] * 3
    L.phx_kv4_page_bytes.restype = _sz
    L.phx_kv4_append.argtypes = [_vp, _cache, _batch, ctypes.c_int, _u64, _u64, _i64, _i64]
    L.phx_kv4_read.argtypes = L.phx_kv4_append.argtypes
    L.phx_kv4_attention.argtypes = [_vp, _cache, _batch, ctypes.c_int, _u64, _u64, _i64,
                                    ctypes.c_float, ctypes.c_int, _i64, _i64]
    _f8, _f8w = ctypes.POINTER(F8Rows), ctypes.POINTER(F8Weights)
    L.phx_norm_f8.argtypes = [_vp, ctypes.c_int] + [_u64] * 5 + [_f8, _i64, _i64, ctypes.c_float] + \
        [_i64] * 4
    L.phx_glu_f8.argtypes = [_vp, ctypes.c_int, _u64, _f8, _i64]
    L.phx_gemm_f8.argtypes = [_vp, _f8, _f8w, ctypes.c_int, _u64, ctypes.c_float, ctypes.c_float, _i64]
    L.phx_gemm_f8_grouped.argtypes = [_vp, _f8, _f8w, _u64, _u64, _i64, ctypes.c_int, _u64,
                                      ctypes.c_float, ctypes.c_float, _i64]
    L.phx_kv4_split_plan.argtypes = [_cache, _batch, _i64, ctypes.POINTER(ctypes.c_int),
                                     ctypes.POINTER(_sz)]
    _pi64, _pi32 = ctypes.POINTER(_i64), ctypes.POINTER(ctypes.c_int32)
    L.phx_pages_create.argtypes = [ctypes.POINTER(_vp), ctypes.c_int32, ctypes.c_int32]
    L.phx_pages_destroy.argtypes = [_vp]
    L.phx_pages_new.argtypes = [_vp, _pi64]
    L.phx_pages_resize.argtypes = [_vp, _i64, _i64]
    L.phx_pages_fork.argtypes = [_vp, _i64, _pi64]
    L.phx_pages_free.argtypes = [_vp, _i64]
    L.phx_pages_compact.argtypes = [_vp]
    L.phx_pages_table.argtypes = [_vp, _i64, _pi32, _i64, _pi64]
    L.phx_pages_stats.argtypes = [_vp, _pi64, _pi64, _pi64]
    L.phx_pages_pending.argtypes = [_vp, _pi32, _pi32, _i64, _pi64, ctypes.c_int]
    L.phx_pages_apply.argtypes = [_vp, _vp, _u64, _sz, _i64, _u64]
    L.phx_pages_copy.argtypes = [_vp, _u64, _i64, _sz, _vp, _vp, _i64, _i64, _u64]
    L.phx_size_class.argtypes = [_sz]
    L.phx_size_class.restype = _sz
    L.phx_arena_create.argtypes = [ctypes.POINTER(_vp), _sz]
    L.phx_arena_destroy.argtypes = [_vp]
    L.phx_arena_alloc.argtypes = [_vp, _sz, ctypes.POINTER(_u64), ctypes.POINTER(_sz)]
    L.phx_arena_free.argtypes = [_vp, _u64, _sz]
    L.phx_arena_can_alloc.argtypes = [_vp, _sz]
    L.phx_arena_stats.argtypes = [_vp, ctypes.POINTER(_sz), ctypes.POINTER(_sz),
                                  ctypes.POINTER(_u64)]
    L.phx_lcg_fill_f32.argtypes = [_u64, _sz, ctypes.POINTER(ctypes.c_float)]
    L.phx_normal_fill_f32.argtypes = [_u64, _sz, ctypes.c_double, ctypes.POINTER(ctypes.c_float)]
    L.phx_f32_to_f16.argtypes = [_sz, ctypes.POINTER(ctypes.c_float),
                                 ctypes.POINTER(ctypes.c_uint16)]
    L.phx_f16_to_f32.argtypes = [_sz, ctypes.POINTER(ctypes.c_uint16),
                                 ctypes.POINTER(ctypes.c_float)]
    L.phx_pod_create.argtypes = [ctypes.POINTER(_vp), _sz, ctypes.c_int]
    L.phx_pod_destroy.argtypes = [_vp]
    L.phx_pod_get_arena.argtypes = [_vp, ctypes.POINTER(_vp)]
    L.phx_pod_set_tensor.argtypes = [_vp, ctypes.c_uint32, ctypes.c_char_p,
                                     ctypes.POINTER(_u64), ctypes.c_uint32]
    L.phx_pod_set_kernel.argtypes = [_vp, ctypes.c_uint32, ctypes.c_int]
    L.phx_pod_set_kernel_function.argtypes = [_vp, ctypes.c_uint32, _vp, ctypes.c_int]
    L.phx_pod_run_segment.argtypes = [_vp, ctypes.c_char_p, ctypes.POINTER(_u64)]
    L.phx_lcg_fill_f32_stream.argtypes = [ctypes.POINTER(_u64), ctypes.c_size_t, _vp]
    L.phx_pod_set_manifest_pb.argtypes = [_vp, ctypes.c_char_p, ctypes.c_size_t]
    L.phx_pod_run_segment_pb.argtypes = [_vp, ctypes.c_char_p, ctypes.c_size_t,
                                         ctypes.POINTER(_u64)]
    L.phx_segment_pb_to_text.argtypes = [ctypes.c_char_p, ctypes.c_size_t, ctypes.c_char_p,
                                         ctypes.c_size_t, ctypes.POINTER(ctypes.c_size_t)]
    _LIB = L
    return L


def check(rc):
    if rc != 0:
        raise PhxError(rc, lib().phx_last_error().decode(errors="replace"))


def init(device=0):
    """cust::quick_init (main.rs:169): select the device and load code objects lazily."""
    global _INIT
    if not _INIT:
        code_dir = os.environ.get("PHX_CODE_OBJECT_DIR") or LIB_DIR
        check(lib().phx_init(device, code_dir.encode()))
        _INIT = True


def device_info():
    name = ctypes.create_string_buffer(256)
    cus, clk, lds = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    hbm = _sz()
    check(lib().phx_device_info(name, 256, ctypes.byref(cus), ctypes.byref(clk),
                                ctypes.byref(hbm), ctypes.byref(lds)))
    return {"name": name.value.decode(), "cus": cus.value, "clock_khz": clk.value,
            "hbm_bytes": hbm.value, "lds_bytes_per_cu": lds.value}


def synchronize():
    check(lib().phx_device_synchronize())


# ------------------------------------------------------------------- memory
class DeviceBuffer:
    """A hipMalloc'd buffer (the reference's DeviceBuffer / as_dbuf)."""

    def __init__(self, nbytes):
        self.nbytes = int(nbytes)
        p = _u64()
        check(lib().phx_malloc(ctypes.byref(p), self.nbytes))
        self.ptr = p.value

    @classmethod
    def from_array(cls, arr):
        arr = np.ascontiguousarray(arr)
        b = cls(arr.nbytes)
        b.upload(arr)
        return b

    def upload(self, arr):
        arr = np.ascontiguousarray(arr)
        assert arr.nbytes <= self.nbytes
        check(lib().phx_memcpy_h2d(self.ptr, arr.ctypes.data, arr.nbytes))

    def download(self, dtype, shape):
        out = np.empty(shape, dtype)
        assert out.nbytes <= self.nbytes
        check(lib().phx_memcpy_d2h(out.ctypes.data, self.ptr, out.nbytes))
        return out

    def zero(self, stream=None):
        check(lib().phx_memset_async(self.ptr, 0, self.nbytes, _sh(stream)))

    def free(self):
        if self.ptr:
            check(lib().phx_free(self.ptr))
            self.ptr = 0

    def __del__(self):
        try:
            if self.ptr and _LIB is not None:
                _LIB.phx_free(self.ptr)
                self.ptr = 0
        except Exception:
            pass


class Stream:
    """A non-blocking HIP stream at default priority (main.rs:170)."""

    def __init__(self):
        h = _vp()
        check(lib().phx_stream_create(ctypes.byref(h)))
        self.handle = h.value

    def synchronize(self):
        check(lib().phx_stream_synchronize(self.handle))

    def destroy(self):
        if self.handle:
            check(lib().phx_stream_destroy(self.handle))
            buf = _WORKSPACES.pop(self.handle, None)
            if buf is not None:
                buf.free()  # the stream was drained by its destroy
            self.handle = None


class Event:
    def __init__(self):
        h = _vp()
        check(lib().phx_event_create(ctypes.byref(h)))
        self.handle = h.value

    def record(self, stream):
        check(lib().phx_event_record(self.handle, stream.handle if stream else None))

    def synchronize(self):
        check(lib().phx_event_synchronize(self.handle))

    def query(self):
        rc = lib().phx_event_query(self.handle)
        if rc not in (0, 1):
            check(rc)
        return rc == 0

    def elapsed_ms(self, later):
        ms = ctypes.c_float()
        check(lib().phx_event_elapsed_ms(ctypes.byref(ms), self.handle, later.handle))
        return ms.value

    def destroy(self):
        if self.handle:
            check(lib().phx_event_destroy(self.handle))
            self.handle = None


def _sh(stream):
    return stream.handle if isinstance(stream, Stream) else stream


# Workspaces bound by bind_workspace, kept alive while bound: stream handle -> buffer
_WORKSPACES = {}


def set_workspace(stream, addr, nbytes):
    """phx_stream_set_workspace: bind caller-owned device memory (256-byte
    aligned) as the split workspace of launches on stream (None: the legacy
    default stream); addr 0 unbinds.  The caller keeps the memory alive."""
    check(lib().phx_stream_set_workspace(_sh(stream), int(addr), int(nbytes)))


def get_workspace(stream):
    """(address, bytes) of the workspace bound to stream, (0, 0) for none."""
    a, n = _u64(), _sz()
    check(lib().phx_stream_get_workspace(_sh(stream), ctypes.byref(a), ctypes.byref(n)))
    return a.value, n.value


def bind_workspace(stream, nbytes):
    """Allocates a workspace of nbytes (hipMalloc, 256-byte aligned) and binds
    it to stream, replacing (and freeing) one an earlier call bound; nbytes 0
    unbinds.  Split launches on the stream then use it; the launches
    themselves never allocate."""
    key = _sh(stream)
    set_workspace(stream, 0, 0)
    old = _WORKSPACES.pop(key, None)
    if old is not None:
        synchronize()  # launches in flight may still use it
        old.free()
    if nbytes:
        buf = DeviceBuffer(nbytes)
        set_workspace(stream, buf.ptr, nbytes)
        _WORKSPACES[key] = buf


# ------------------------------------------------------------------- launches
def _addr(buf, nbytes, what):
    """Device address of `buf` (a DeviceBuffer or a raw address).  For a
    DeviceBuffer the size is checked against the bytes the kernel touches, so
    a wrong buffer raises on the host instead of faulting the GPU."""
    if type(buf) is int:
        return buf
    if isinstance(buf, DeviceBuffer):
        if buf.nbytes < nbytes:
            raise PhxError(PHX_E_INVALID, f"{what}: buffer holds {buf.nbytes} B, kernel "
                                          f"accesses {nbytes} B")
        return buf.ptr
    return int(buf)


# gemm_fp32's tilings by launch-plan variant (TILE_M, TILE_N, TILE_K), as
# include/phobos_hip.h lists them; variant 0 is the built-in tiling.
GEMM_FP32_TILINGS = [(256, 256, 16), (256, 128, 16), (128, 256, 16), (128, 128, 16),
                     (128, 128, 32), (128, 128, 8), (256, 256, 8), (64, 64, 16)]

_GEMM_ESZ = {GEMM_FP32: 4, GEMM_FP16TC_FP32ACC: 4, GEMM_FP16: 2, MATMUL: 4}


def launch_saxpy(stream, x, y, out, n, alpha):
    """saxpy_fp32.ph: out = alpha*x + y (main.rs:1227-1239)."""
    check(lib().phx_saxpy(_sh(stream), _addr(x, 4 * n, "x"), _addr(y, 4 * n, "y"),
                          _addr(out, 4 * n, "out"), n, alpha))


def launch_gemm(stream, kernel, a, b, c, M, N, K, alpha, beta):
    """C = alpha*A@B + beta*C for the gemm-family kernel ids (main.rs:290-327)."""
    e = _GEMM_ESZ.get(kernel, 4)
    check(lib().phx_gemm(_sh(stream), kernel, _addr(a, e * M * K, "A"), _addr(b, e * K * N, "B"),
                         _addr(c, e * M * N, "C"), M, N, K, alpha, beta))


def launch_matmul_init(stream, c, M, N, beta):
    check(lib().phx_matmul_init(_sh(stream), _addr(c, 4 * M * N, "C"), M, N, beta))


def launch_flash(stream, kernel, q, k, v, o, Nq, Nk, D, scale):
    """One-head flash attention (main.rs:334-371)."""
    e = 2 if kernel == FLASH_FP16 else 4
    check(lib().phx_flash_attention(_sh(stream), kernel, _addr(q, e * Nq * D, "Q"),
                                    _addr(k, e * Nk * D, "K"), _addr(v, e * Nk * D, "V"),
                                    _addr(o, e * Nq * D, "O"), Nq, Nk, D, scale))


def launch_flash_bh(stream, kernel, q, k, v, o, BH, Nq, Nk, D, scale):
    e = 2 if kernel == FLASH_FP16_BH else 4
    check(lib().phx_flash_attention_bh(_sh(stream), kernel, _addr(q, e * BH * Nq * D, "Q"),
                                       _addr(k, e * BH * Nk * D, "K"),
                                       _addr(v, e * BH * Nk * D, "V"),
                                       _addr(o, e * BH * Nq * D, "O"), BH, Nq, Nk, D, scale))


# ------------------------------------------------------------------- decode operators
_ESZ = {F32: 4, F16: 2}


def _span(rows, ld, width, esz):
    """Bytes from the first to past the last of `rows` rows, ld elements apart."""
    return ((rows - 1) * (ld or width) + width) * esz if rows else 0


def w4_packed_bytes(N, K):
    return lib().phx_w4_packed_bytes(N, K)


def w4_pack(stream, codes, packed, N, K):
    """Codes u8 [K, N] (0 .. 15) into the tiles launch_gemv_w4 reads."""
    check(lib().phx_w4_pack(_sh(stream), _addr(codes, N * K, "codes"),
                            _addr(packed, w4_packed_bytes(N, K), "packed"), N, K))


def w4_quantize(b, group):
    """Codes u8 [K, N], scales f16 and zero points u8 [ceil(K/group), N] of
    weights b [K, N]: each group's range, widened to hold 0, in 15 steps, so
    that a weight of 0 stays 0.  Host arrays."""
    b = np.asarray(b, np.float64)
    K, N = b.shape
    groups = -(-K // group)
    padded = np.zeros((groups * group, N))
    padded[:K] = b
    padded = padded.reshape(groups, group, N)
    lo, hi = np.minimum(padded.min(1), 0), np.maximum(padded.max(1), 0)
    with np.errstate(over="ignore", invalid="ignore"):
        scales = ((hi - lo) / 15).astype(np.float16)
    if not np.isfinite(scales).all():
        raise PhxError(PHX_E_INVALID, "w4_quantize: weights that are infinite or NaN, or a range of more "
                       "than 15 * 65504")
    # below 2^-14 f16 numbers are 2^-24 apart: one too small leaves a weight out of reach
    short = (scales < np.float16(2.0 ** -14)) & (scales.astype(np.float64) < (hi - lo) / 15)
    scales = np.where(short, np.nextafter(scales, np.float16(1)), scales)
    scales = np.where(scales > 0, scales, np.float16(2.0 ** -24))
    s = scales.astype(np.float64)
    zeros = np.clip(np.rint(-lo / s), 0, 15)
    codes = np.clip(np.rint(padded / s[:, None]) + zeros[:, None], 0, 15)
    return (codes.reshape(-1, N)[:K].astype(np.uint8), scales, zeros.astype(np.uint8))


def launch_gemv_w4(stream, dtype, a, w, scales, zeros, c, M, N, K, group, alpha=1.0, beta=0.0,
                   lda=0, ldc=0):
    """C = alpha*A@W + beta*C, up to 64 rows, 4-bit weights (phx_gemv_w4);
    zeros 0 for zero points of 8."""
    e, g = _ESZ.get(dtype, 4), -(-K // group) if group > 0 else 0
    check(lib().phx_gemv_w4(_sh(stream), dtype, _addr(a, _span(M, lda, K, e), "A"),
                            _addr(w, w4_packed_bytes(N, K), "W"), _addr(scales, 2 * g * N, "scales"),
                            _addr(zeros, g * N, "zeros"), _addr(c, _span(M, ldc, N, e), "C"),
                            M, N, K, group, alpha, beta, lda, ldc))


def kv4_page_bytes(heads, head_dim, page_tokens):
    if not _fit32(heads, head_dim, page_tokens):
        return 0
    return lib().phx_kv4_page_bytes(heads, head_dim, page_tokens)


def launch_kv4_append(stream, cache, batch, dtype, k, v, ldk=0, ldv=0):
    """The rows' K and V [rows][heads][head_dim], quantised, into the cache
    (phx_kv4_append)."""
    e, w = _ESZ.get(dtype, 4), cache.heads * cache.head_dim
    check(lib().phx_kv4_append(_sh(stream), cache, batch, dtype,
                               _addr(k, _span(batch.rows, ldk, w, e), "K"),
                               _addr(v, _span(batch.rows, ldv, w, e), "V"), ldk, ldv))


def launch_kv4_read(stream, cache, batch, dtype, k, v, ldk=0, ldv=0):
    """The rows' K and V as the cache holds them (phx_kv4_read)."""
    e, w = _ESZ.get(dtype, 4), cache.heads * cache.head_dim
    check(lib().phx_kv4_read(_sh(stream), cache, batch, dtype,
                             _addr(k, _span(batch.rows, ldk, w, e), "K"),
                             _addr(v, _span(batch.rows, ldv, w, e), "V"), ldk, ldv))


def launch_kv4_attention(stream, cache, batch, dtype, q, o, q_heads, scale, causal=True, ldq=0,
                         ldo=0):
    """Attention of the rows' queries over their sequences in the cache
    (phx_kv4_attention)."""
    e, w = _ESZ.get(dtype, 4), q_heads * cache.head_dim
    check(lib().phx_kv4_attention(_sh(stream), cache, batch, dtype,
                                  _addr(q, _span(batch.rows, ldq, w, e), "Q"),
                                  _addr(o, _span(batch.rows, ldo, w, e), "O"), q_heads, scale,
                                  1 if causal else 0, ldq, ldo))


def kv4_split_plan(cache, batch, q_heads):
    """(splits, workspace bytes) of such an attention (phx_kv4_split_plan)."""
    sp, ws = ctypes.c_int(), _sz()
    check(lib().phx_kv4_split_plan(cache, batch, q_heads, ctypes.byref(sp), ctypes.byref(ws)))
    return sp.value, ws.value


def f8_quantize(w):
    """Codes u8 [..., N, K] (e4m3) and scales f32 [..., ceil(N/128), ceil(K/128)] of
    weights w [..., N, K], K next to each other as F8Weights has them: the largest
    magnitude of each 128 x 128 has the code 448 or -448.  Host arrays."""
    w = np.asarray(w, np.float64)
    if w.ndim < 2 or not w.size:
        raise PhxError(PHX_E_INVALID, f"f8_quantize: weights [..., N, K], got {w.shape}")
    *lead, N, K = w.shape
    nb, kb = -(-N // 128), -(-K // 128)
    b = np.zeros((*lead, nb * 128, kb * 128))
    b[..., :N, :K] = w
    b = b.reshape(*lead, nb, 128, kb, 128)
    a = np.abs(b).max((-3, -1))
    with np.errstate(over="ignore"):
        scales = (a / 448).astype(np.float32)
    # (below 2^-126 an f32 scale keeps few bits, or none)
    if not np.isfinite(scales).all() or (scales[a > 0] < 2.0 ** -126).any():
        raise PhxError(PHX_E_INVALID, "f8_quantize: weights that are infinite or NaN, or that no f32 "
                       "scale holds")
    q = b * 448 / np.where(a > 0, a, 1)[..., :, None, :, None]
    step = np.exp2(np.floor(np.log2(np.maximum(np.abs(q), 2.0 ** -6))) - 3)
    q = np.rint(q / step) * step  # ties to even, as every rounding to e4m3
    exponent = np.floor(np.log2(np.maximum(np.abs(q), 2.0 ** -6)))
    # steps of 2^-9 from 0, of which each power of two from 2^-6 on takes eight
    code = np.abs(q) / np.exp2(exponent - 3) + (exponent + 6) * 8
    code = code.astype(np.uint8) | (np.signbit(q).astype(np.uint8) << 7)
    return np.ascontiguousarray(code.reshape(*lead, nb * 128, kb * 128)[..., :N, :K]), scales


def launch_norm_f8(stream, dtype, x, r, gain, h, y, q, M, K, eps, ldx=0, ldr=0, ldh=0, ldy=0):
    """The root-mean-square norm of X + R (r 0: of X), which goes to H, times the
    gain: in 8 bits to q (F8Rows or None) and as it is to Y (0: not wanted)
    (phx_norm_f8)."""
    # (raw addresses are nothing to be looked at, and that takes 1 us of 5)
    if not (type(x) is type(r) is type(gain) is type(h) is type(y) is int):
        e = _ESZ.get(dtype, 4)
        x, r = _addr(x, _span(M, ldx, K, e), "X"), _addr(r, _span(M, ldr, K, e), "R")
        gain = _addr(gain, K * e, "gain")
        h, y = _addr(h, _span(M, ldh, K, e), "H"), _addr(y, _span(M, ldy, K, e), "Y")
    check(lib().phx_norm_f8(_sh(stream), dtype, x, r, gain, h, y, q, M, K, eps, ldx, ldr, ldh, ldy))


def launch_glu_f8(stream, dtype, u, q, ldu=0):
    """silu(gate) * value of rows U [gates | values] into the 8-bit rows q
    (phx_glu_f8)."""
    if type(u) is not int and q:
        u = _addr(u, _span(q.rows, ldu, 2 * q.k, _ESZ.get(dtype, 4)), "U")
    check(lib().phx_glu_f8(_sh(stream), dtype, u, q, ldu))


def launch_gemm_f8(stream, a, w, dtype, c, alpha=1.0, beta=0.0, ldc=0):
    """C = alpha*A@W^T + beta*C of 8-bit rows and weights (phx_gemm_f8)."""
    if type(c) is not int and a and w:
        c = _addr(c, _span(a.rows, ldc, w.n, _ESZ.get(dtype, 4)), "C")
    check(lib().phx_gemm_f8(_sh(stream), a, w, dtype, c, alpha, beta, ldc))


def launch_gemm_f8_grouped(stream, a, w, starts, order, M, dtype, c, alpha=1.0, beta=0.0, ldc=0):
    """The same for M rows sorted by expert: rows starts[e] up to starts[e+1] of C
    are A's rows order[i] (order 0: A's own) times expert e's weights
    (phx_gemm_f8_grouped)."""
    if not (type(starts) is type(order) is type(c) is int) and w:
        starts, order = _addr(starts, 4 * (w.experts + 1), "starts"), _addr(order, 4 * M, "order")
        c = _addr(c, _span(M, ldc, w.n, _ESZ.get(dtype, 4)), "C")
    check(lib().phx_gemm_f8_grouped(_sh(stream), a, w, starts, order, M, dtype, c, alpha, beta, ldc))


def _page_list(x):
    """x, whole numbers of any kind, as an i32 array of its own."""
    if getattr(x, "dtype", None) == np.int32:
        x = np.array(x, np.int32)
    else:
        try:
            x = list(x.tolist() if hasattr(x, "tolist") else x)
            if x and isinstance(x[0], bool):
                raise TypeError("a mask is no list of page numbers")
            # array() takes whole numbers alone, and those that fit
            x = np.frombuffer(array.array("i", x), np.int32) if x else np.empty(0, np.int32)
        except (TypeError, OverflowError) as e:
            raise PhxError(PHX_E_INVALID, f"pages_copy: {e}") from None
    if x.ndim != 1:
        raise PhxError(PHX_E_INVALID, "pages_copy: src and dst are lists of page numbers")
    return x


def _layers(pool, pages, page_bytes, layers, layer_stride):
    """The address of `layers` pools of pages."""
    whole = (layers - 1) * layer_stride + pages * page_bytes if layers > 0 else 0
    return _addr(pool, whole, "pool")


def pages_copy(stream, pool, pages, page_bytes, src, dst, layers=1, layer_stride=0):
    """Copies page src[i] to page dst[i] in each layer's pool (phx_pages_copy)."""
    src, dst = _page_list(src), _page_list(dst)
    if src.size != dst.size:
        raise PhxError(PHX_E_INVALID, "pages_copy: src and dst are lists of one length")
    # (x.ctypes.data takes four times as long)
    at = [ctypes.byref(ctypes.c_int32.from_buffer(x)) if x.size else None for x in (src, dst)]
    check(lib().phx_pages_copy(_sh(stream), _layers(pool, pages, page_bytes, layers, layer_stride),
                               pages, page_bytes, *at, src.size, layers, layer_stride))


class Pages:
    """Which page of a cache belongs to which sequence (phx_pages_*)."""

    def __init__(self, pages, page_tokens):
        self.handle = None
        h = _vp()
        if not _fit32(pages, page_tokens):
            raise PhxError(PHX_E_INVALID, f"pages_create: {pages} pages of {page_tokens} tokens")
        check(lib().phx_pages_create(ctypes.byref(h), pages, page_tokens))
        self.handle, self.pages = h.value, pages

    def new(self):
        seq = _i64()
        check(lib().phx_pages_new(self.handle, ctypes.byref(seq)))
        return seq.value

    def resize(self, seq, tokens):
        check(lib().phx_pages_resize(self.handle, seq, tokens))

    def fork(self, seq):
        child = _i64()
        check(lib().phx_pages_fork(self.handle, seq, ctypes.byref(child)))
        return child.value

    def free(self, seq):
        check(lib().phx_pages_free(self.handle, seq))

    def compact(self):
        check(lib().phx_pages_compact(self.handle))

    def table(self, seq):
        n, cap = _i64(), 0
        while True:  # other threads may change it between its size and its contents
            out = np.empty(cap, np.int32)
            check(lib().phx_pages_table(self.handle, seq,
                                        out.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), cap,
                                        ctypes.byref(n)))
            if n.value <= cap:
                return out[:n.value]
            cap = n.value

    def stats(self):
        """(pages in use, one past the highest of them, pending copies)."""
        v = [_i64() for _ in range(3)]
        check(lib().phx_pages_stats(self.handle, *(ctypes.byref(x) for x in v)))
        return tuple(x.value for x in v)

    def pending(self, clear=False):
        """The pending copies as (src, dst) arrays; with clear the caller runs
        them and they are no longer pending."""
        n, cap = _i64(), self.stats()[2]
        while True:  # as table()
            out = [np.empty(cap, np.int32) for _ in range(2)]
            ptr = [x.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)) for x in out]
            rc = lib().phx_pages_pending(self.handle, *ptr, cap, ctypes.byref(n), 1 if clear else 0)
            if n.value <= cap:
                check(rc)
                return tuple(x[:n.value] for x in out)
            cap = n.value

    def apply(self, stream, pool, page_bytes, layers=1, layer_stride=0):
        """Launches the pending copies in the layers' pools and clears them."""
        check(lib().phx_pages_apply(self.handle, _sh(stream),
                                    _layers(pool, self.pages, page_bytes, layers, layer_stride),
                                    page_bytes, layers, layer_stride))

    def destroy(self):
        if self.handle:
            check(lib().phx_pages_destroy(self.handle))
            self.handle = None

    def __del__(self):
        try:
            if self.handle and _LIB is not None:
                _LIB.phx_pages_destroy(self.handle)
                self.handle = None
        except Exception:
            pass


def grid_for(kernel, dims):
    d = (_i64 * len(dims))(*dims)
    g, b = _u32a3(), _u32a3()
    check(lib().phx_grid_for(kernel, d, len(dims), g, b))
    return tuple(g), tuple(b)


def kernel_by_name(ph_file, entry):
    """Built-in kernel id for the reference's .ph file stem and entry name."""
    k = ctypes.c_int()
    check(lib().phx_kernel_by_name(ctypes.byref(k), ph_file.encode(), entry.encode()))
    return k.value


def check_shape(kernel, dims):
    d = (_i64 * len(dims))(*dims)
    return lib().phx_check_shape(kernel, d, len(dims))


def split_plan(kernel, dims):
    """(splits, workspace bytes) of a launch of kernel over dims (phx_split_plan)."""
    d = (_i64 * len(dims))(*dims)
    sp, ws = ctypes.c_int(), _sz()
    check(lib().phx_split_plan(kernel, d, len(dims), ctypes.byref(sp), ctypes.byref(ws)))
    return sp.value, ws.value


class Plan(ctypes.Structure):
    """phx_plan: K or key chunks (1 = unsplit) and kernel variant."""
    _fields_ = [("splits", ctypes.c_int32), ("variant", ctypes.c_int32)]


def plan_get(kernel, dims):
    """(splits, variant) a launch of kernel over dims uses now (phx_plan_get)."""
    d = (_i64 * len(dims))(*dims)
    p = Plan()
    check(lib().phx_plan_get(kernel, d, len(dims), ctypes.byref(p)))
    return p.splits, p.variant


def plan_pin(kernel, dims, splits=None, variant=0):
    """Pins (splits, variant) for kernel at dims; splits None removes the pin."""
    d = (_i64 * len(dims))(*dims)
    p = None if splits is None else ctypes.byref(Plan(splits, variant))
    check(lib().phx_plan_pin(kernel, d, len(dims), p))


def plan_unpin_all():
    check(lib().phx_plan_unpin_all())


def kernel_abi(kernel):
    bits = ctypes.c_int()
    b = _u32a3()
    check(lib().phx_kernel_abi(kernel, ctypes.byref(bits), b))
    return bits.value, tuple(b)


def builtin_function(kernel):
    f = _vp()
    check(lib().phx_builtin_function(ctypes.byref(f), kernel))
    return f.value


def module_load_data(image):
    """PtxCache::insert with a gfx950 code object in place of PTX
    (phobos-pod/src/ptx_cache.rs:12-82): returns a module handle."""
    m = _vp()
    check(lib().phx_module_load_data(ctypes.byref(m), image, len(image)))
    return m.value


def module_get_function(module, name):
    f = _vp()
    check(lib().phx_module_get_function(ctypes.byref(f), module, name.encode()))
    return f.value


def module_unload(module):
    check(lib().phx_module_unload(module))


def compute(func, index_bits, tiles, scalars, grid, cta, stream=None):
    """Pod COMPUTE marshalling (engine.rs:582-647).

    tiles: [(addr, shape_tuple)], scalars: [(pos, bytes, bits)]."""
    ta = (TileArg * max(1, len(tiles)))()
    for i, (addr, shape) in enumerate(tiles):
        ta[i].addr = addr
        ta[i].rank = len(shape)
        for j, s in enumerate(shape):
            ta[i].shape[j] = s
    sa = (ScalarArg * max(1, len(scalars)))()
    for i, (pos, nbytes, bits) in enumerate(scalars):
        sa[i].pos, sa[i].bytes, sa[i].bits = pos, nbytes, bits
    check(lib().phx_compute(func, index_bits, ta, len(tiles), sa, len(scalars), _u32a3(*grid),
                            _u32a3(*cta), _sh(stream)))


def f32_bits(x):
    """ScalarValue::F32(x).to_bits() (phobos-cluster/src/tile.rs:75-84)."""
    return int(np.array([x], np.float32).view(np.uint32)[0])


# ------------------------------------------------------------------- inputs
def lcg_f32(seed, n):
    """Lcg::unit_f32s (phobos-base/src/rng.rs:9-25), generated by the library."""
    out = np.empty(n, np.float32)
    check(lib().phx_lcg_fill_f32(seed, n, out.ctypes.data_as(ctypes.POINTER(ctypes.c_float))))
    return out


def normal_f32(seed, n, scale=1.0):
    out = np.empty(n, np.float32)
    check(lib().phx_normal_fill_f32(seed, n, scale,
                                    out.ctypes.data_as(ctypes.POINTER(ctypes.c_float))))
    return out


def to_f16_bits(x):
    x = np.ascontiguousarray(x, np.float32)
    out = np.empty(x.shape, np.uint16)
    check(lib().phx_f32_to_f16(x.size, x.ctypes.data_as(ctypes.POINTER(ctypes.c_float)),
                               out.ctypes.data_as(ctypes.POINTER(ctypes.c_uint16))))
    return out


def from_f16_bits(bits):
    bits = np.ascontiguousarray(bits, np.uint16)
    out = np.empty(bits.shape, np.float32)
    check(lib().phx_f16_to_f32(bits.size, bits.ctypes.data_as(ctypes.POINTER(ctypes.c_uint16)),
                               out.ctypes.data_as(ctypes.POINTER(ctypes.c_float))))
    return out


def segment_pb_to_text(data):
    """Decodes an encoded phobos.v1.Segment into the pod's text form
    (phx_segment_pb_to_text; no device needed)."""
    need = ctypes.c_size_t()
    check(lib().phx_segment_pb_to_text(data, len(data), None, 0, ctypes.byref(need)))
    buf = ctypes.create_string_buffer(need.value)
    check(lib().phx_segment_pb_to_text(data, len(data), buf, need.value, ctypes.byref(need)))
    return buf.value.decode()
