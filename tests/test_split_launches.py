"""The two launches of a split call (its parts, and what joins them) share the
stream's workspace: no other thread's launch on the stream may come between.
Against a recording stand-in for the HIP runtime (fake_hip.c), without a GPU."""
import os
import shutil
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))

_CHILD = """
import ctypes, sys, threading
class Launch(ctypes.Structure):
    _fields_ = [("stream", ctypes.c_void_p), ("name", ctypes.c_char * 64), ("thread", ctypes.c_uint64)]
fake = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
fake.fake_launch.restype = ctypes.POINTER(Launch)
sys.path[:0] = [sys.argv[2]]
import phobos_amd as px
px.init(0)
A = 1 << 20
s = px.Stream()
px.set_workspace(s, A, 1 << 30)
cache = px.Kv4Cache(A, 500, 1, 64, 64)
batch = px.Kv4Batch(A, 200, A, 0, 1, 1, 9000, 1)
calls = [
    lambda: px.launch_gemm(s, px.GEMM_FP16TC_FP32ACC, A, A, A, 256, 256, 8192, 1.0, 0.0),
    lambda: px.launch_gemm(s, px.GEMM_FP32, A, A, A, 64, 64, 8192, 1.0, 0.0),
    lambda: px.launch_flash(s, px.FLASH_FP16, A, A, A, A, 4096, 4096, 64, 0.125),
    lambda: px.launch_flash_bh(s, px.FLASH_FP32_BH, A, A, A, A, 1, 512, 8192, 64, 0.125),
    lambda: px.launch_gemv_w4(s, px.F16, A, A, A, 0, A, 40, 1500, 8192, 32),
    lambda: px.launch_kv4_attention(s, cache, batch, px.F16, A, A, 4, 0.125),
]
for f in calls:  # each is two launches
    n = fake.fake_count()
    f()
    assert fake.fake_count() == n + 2, (calls.index(f), fake.fake_count() - n)
first = fake.fake_count()
threads = [threading.Thread(target=lambda f=f: [f() for _ in range(15)]) for f in calls]
[t.start() for t in threads]
[t.join() for t in threads]
log = [fake.fake_launch(i).contents for i in range(first, fake.fake_count())]
assert len(log) == 2 * 15 * len(calls)
for a, b in zip(log[::2], log[1::2]):
    names = a.name.decode(), b.name.decode()
    assert a.thread == b.thread, ("apart", names)
    assert "reduce" in names[1] or "combine" in names[1], names
print("kept together", len({a.thread for a in log}))
"""


@pytest.mark.parametrize("env", [{}, {"PHX_GEMM_SPLIT": "3", "PHX_FLASH_SPLIT": "3"}])
def test_the_launches_of_a_split_call_stay_together(tmp_path, env):
    cc = shutil.which("cc") or shutil.which("gcc")
    if not cc:
        pytest.skip("no C compiler")
    so = str(tmp_path / "libfake_hip.so")
    subprocess.run([cc, "-shared", "-fPIC", "-O1", "-D_GNU_SOURCE", "-o", so,
                    os.path.join(HERE, "fake_hip.c"), "-lpthread"], check=True)
    out = subprocess.run([sys.executable, "-c", _CHILD, so,
                          os.path.join(os.path.dirname(HERE), "phobos-lang_amd")],
                         capture_output=True, text=True, timeout=120, env=dict(os.environ, **env))
    assert out.stdout.strip() == "kept together 6", out.stderr[-2000:]
