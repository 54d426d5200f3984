"""Which kernels the operators over 8-bit rows and weights launch: every one that is
built is taken by a shape that the GPU tests run, and no other is asked for.
Against a recording stand-in for the HIP runtime (fake_hip.c), without a GPU."""
import os
import re
import shutil
import subprocess
import sys

import pytest

import phobos_amd as px
import test_gpu_f8_rows
import test_gpu_gemm_f8 as gemm

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
shapes, grouped, lengths = json.loads(sys.argv[3])
for t in (px.F16, px.F32):
    for M, N, K in shapes:
        px.launch_gemm_f8(s, px.F8Rows(A, A, M, K), px.F8Weights(A, A, 1, N, K), t, A)
    for M, E, N, K in grouped:
        px.launch_gemm_f8_grouped(s, px.F8Rows(A, A, M, K), px.F8Weights(A, A, E, N, K), A, 0, M, t, A)
    for K in lengths:
        px.launch_norm_f8(s, t, A, A, A, A, 0, px.F8Rows(A, A, 3, K), 3, K, 1e-5)
    px.launch_glu_f8(s, t, A, px.F8Rows(A, A, 3, 64))
print("\\n".join(fake.fake_launch(i).contents.name.decode() for i in range(fake.fake_count())))
"""


def test_every_kernel_is_reached(tmp_path):
    import json
    cc = shutil.which("cc") or shutil.which("gcc")
    if not cc:
        pytest.skip("no C compiler")
    so = str(tmp_path / "libfake_hip.so")
    subprocess.run([cc, "-shared", "-fPIC", "-O1", "-D_GNU_SOURCE", "-o", so,
                    os.path.join(HERE, "fake_hip.c"), "-lpthread"], check=True)
    what = [gemm.SHAPES + gemm.LARGE, [g[:4] for g in gemm.GROUPED], test_gpu_f8_rows.LENGTHS]
    out = subprocess.run([sys.executable, "-c", _CHILD, so,
                          os.path.join(os.path.dirname(HERE), "phobos-lang_amd"), json.dumps(what)],
                         capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stderr[-2000:]
    launched = set(out.stdout.split())
    built = set()
    for name in ("f8_rows.hsaco", "gemm_f8.hsaco"):
        with open(os.path.join(px.LIB_DIR, name), "rb") as f:
            built |= {m.decode() for m in re.findall(rb"\0((?:gemm|norm|glu)_f8_[a-z0-9_]+)\.kd", f.read())}
    assert len(built) == 13 + 16
    assert launched == built, (launched - built, built - launched)
