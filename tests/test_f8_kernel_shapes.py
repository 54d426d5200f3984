"""Which kernel each shape of test_gpu_gemm_f8_kernels.py takes, and that every kernel
that is built has its own shapes there: dense and grouped.  Against a recording stand-in
for the HIP runtime (fake_hip.c), without a GPU."""
import json
import os
import re
import shutil
import subprocess
import sys

import pytest

import phobos_amd as px
import test_gpu_gemm_f8_kernels as kernels

HERE = os.path.dirname(os.path.abspath(__file__))

_CHILD = """
import ctypes, json, sys
class Launch(ctypes.Structure):
    _fields_ = [("stream", ctypes.c_void_p), ("name", ctypes.c_char * 64), ("thread", ctypes.c_uint64)]
fake = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
fake.fake_launch.restype = ctypes.POINTER(Launch)
sys.path[:0] = [sys.argv[2]]
import phobos_amd as px
px.init(0)
A, s = 1 << 20, px.Stream()
for name, shape in json.loads(sys.argv[3]):
    t = px.F16 if name.startswith("f16") else px.F32
    if len(shape) == 3:
        M, N, K = shape
        px.launch_gemm_f8(s, px.F8Rows(A, A, M, K), px.F8Weights(A, A, 1, N, K), t, A)
    else:  # (a list of other rows asks for the same kernel)
        M, E, N, K = shape
        px.launch_gemm_f8_grouped(s, px.F8Rows(A, A, M, K), px.F8Weights(A, A, E, N, K), A, 0, M, t, A)
        px.launch_gemm_f8_grouped(s, px.F8Rows(A, A, M // 2 + 1, K), px.F8Weights(A, A, E, N, K), A, A, M, t, A)
print("\\n".join(fake.fake_launch(i).contents.name.decode() for i in range(fake.fake_count())))
"""


def test_every_shape_takes_its_kernel(tmp_path):
    cc = shutil.which("cc") or shutil.which("gcc")
    if not cc:
        pytest.skip("no C compiler")
    so = str(tmp_path / "libfake_hip.so")
    subprocess.run([cc, "-shared", "-fPIC", "-O1", "-D_GNU_SOURCE", "-o", so,
                    os.path.join(HERE, "fake_hip.c"), "-lpthread"], check=True)
    cases = kernels.DENSE + kernels.GROUPED
    out = subprocess.run([sys.executable, "-c", _CHILD, so,
                          os.path.join(os.path.dirname(HERE), "phobos-lang_amd"), json.dumps(cases)],
                         capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stderr[-2000:]
    want = [(f"gemm_f8_{name}", shape) for name, shape in cases for _ in range(len(shape) - 2)]
    got = out.stdout.split()
    assert len(got) == len(want)
    assert not [(g, w) for g, w in zip(got, want) if g != w[0]]


def test_every_kernel_has_shapes():
    with open(os.path.join(px.LIB_DIR, "gemm_f8.hsaco"), "rb") as f:
        built = {m.decode() for m in re.findall(rb"\0gemm_f8_([a-z0-9_]+)\.kd", f.read())}
    assert built == set(kernels.KERNELS)
    for dense, grouped in kernels.KERNELS.values():
        assert dense and grouped
        # more than two rounds of the rows' scales; once more than one of the weights'
        assert min(k for *_, k in dense + grouped) > 8 * 128
    assert all(any(k > 64 * 128 for *_, k in dense) for name, (dense, _) in kernels.KERNELS.items()
               if name != "f16_1x1_2x1_k4_s2")  # (which long K leaves to four stages)
