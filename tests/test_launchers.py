"""What the entry points launch, and what they refuse to launch, on a stand-in for the CUDA runtime (``launch_runtime.cpp``): nothing reaches a GPU."""
import os
import re
import subprocess
import sys
from pathlib import Path

import pytest

from tirocinio_triennale_b200 import _build

pytestmark = pytest.mark.skipif(_build.nvcc_path() is None, reason="needs nvcc")

BEGIN = """
import ctypes as C, sys
sys.path.insert(0, sys.argv[2])
from tirocinio_triennale_b200 import _lib_train
from tirocinio_triennale_b200._lib_train import Heads
fake = C.CDLL(None)
fake.fake_name.restype = C.c_char_p
lib = C.CDLL(sys.argv[1])
_lib_train.declare(lib)
at = C.c_void_p(1 << 20)
big = 1 << 45

def launched(call):
    fake.fake_clear()
    status = call()
    return status, [fake.fake_name(i).decode() for i in range(fake.fake_launches())]

def attention(heads, kv, queries, keys, d, kind=1, batch=1):
    h = lambda n, t: Heads(at, n * t * d, t * d, d)
    return lambda: lib.hc_attention(h(heads, queries), h(kv, keys), h(kv, keys), kind, at, at, batch, heads, kv, queries, keys, d, 0, 0, 1.0, None)

def attention_backward(heads, kv, queries, keys, d, kind=1, batch=1):
    h = lambda n, t: Heads(at, n * t * d, t * d, d)
    return lambda: lib.hc_attention_backward(h(heads, queries), at, h(heads, queries), h(kv, keys), h(kv, keys), kind, at, at, at, at, batch, heads, kv, queries, keys, d, 0, 0, 1.0, at, big, None)
"""


@pytest.fixture(scope="module")
def runtime(tmp_path_factory):
    lib = tmp_path_factory.mktemp("fake") / "libfake_launches.so"
    cuda = Path(_build.nvcc_path()).resolve().parent.parent / "include"
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-I", str(cuda), str(Path(__file__).with_name("launch_runtime.cpp")), "-o", str(lib), "-ldl"], check=True)
    return lib


def run(runtime, calls):
    r = subprocess.run([sys.executable, "-c", BEGIN + calls + "\nprint('done')", str(_build.build_cuda()), str(_build.ROOT)], capture_output=True, text=True, timeout=120,
                       env={**os.environ, "LD_PRELOAD": str(runtime)})
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), r.stdout + r.stderr
    return r.stdout


def test_kernels_that_share_registers_out_have_them(runtime):
    """Warps that take more registers than their CTA was launched with would wait for ever: a kernel that was built with fewer is not launched."""
    calls = """
for registers, allowed in ((72, {"none"}), (88, {"64"}), (96, {"64", "128"})):
    fake.fake_registers(registers)
    for d in (64, 128):
        for kind in (1, 2):
            status, names = launched(attention_backward(4, 2, 300, 300, d, kind))
            ran = [n for n in names if "backward" in n]
            print(registers, d, kind, status, names)
            assert (status == 0) == (str(d) in allowed) and len(ran) == (2 if str(d) in allowed else 0)
        status, names = launched(attention(4, 2, 300, 300, d))
        print(registers, d, status, names)
        assert (status == 0 and len(names) == 1) if d == 128 or registers >= 80 else (status != 0 and not names)
"""
    run(runtime, calls)


def test_registers_that_are_shared_out(tmp_path):
    """As the assembler reports them, of the built source: no fewer than the split counts on."""
    cuda = _build.CSRC / "cuda"
    flags = [f for f in _build.NVCC_FLAGS if f != "-lineinfo"]
    out = subprocess.run([_build.nvcc_path(), *flags, "-Xptxas", "-v", "-I", str(cuda.parent / "include"), "-cubin", str(cuda / "hc_attention.cu"), "-o", str(tmp_path / "cubin")],
                         capture_output=True, text=True, check=True).stderr
    seen = 0
    for entry in out.split("Compiling entry function ")[1:]:
        name, used = entry.split("'")[1], int(re.search(r"Used (\d+) registers", entry).group(1))
        kernel = re.search(r"(hc_attention_kernel|hc_attention_backward_kernel)I\S*?Li(\d+)", name)
        if not kernel or kernel.groups() == ("hc_attention_kernel", "128"):
            continue
        seen += 1
        assert (used + 7) // 8 * 8 >= (80 if kernel.group(2) == "64" else 96), name
    assert seen == 10


def test_sums_of_logits_have_room(runtime, tmp_path):
    """Scratch memory is counted for the tiles that are launched, and a launch that has less is refused."""
    lib = _build.build_cuda()
    exe = tmp_path / "loss_room"
    csrc = _build.CSRC
    subprocess.run([_build.nvcc_path(), *_build.NVCC_FLAGS, "-I", str(csrc / "include"), "-I", str(csrc / "cuda"), str(Path(__file__).with_name("loss_room.cu")), "-o", str(exe),
                    str(lib), str(runtime), "-cudart", "shared", "-Xlinker", "-rpath=%s:%s" % (lib.parent, runtime.parent)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120, env={**os.environ, "LD_PRELOAD": str(runtime)})
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
