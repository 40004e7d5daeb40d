"""The interpreter (deepj_b200/csrc/runtime.cu) over a stand-in for the CUDA runtime and for the kernels (tests/fake_cuda), and what a test needs to drive it."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from deepj_b200 import _lib
from deepj_b200 import build as product_build
from deepj_b200 import compute_graph as cg

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def build(folder):
    """The library under test in `folder`, bound like the real one."""
    nvcc, cuda = product_build._nvcc(), os.path.dirname(os.path.dirname(os.path.realpath(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc")))
    src, inc = os.path.join(ROOT, "deepj_b200", "csrc"), ["-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "deepj_b200", "csrc")]
    a, b, out = (os.path.join(folder, n) for n in ("runtime.o", "standin.o", "libstandin.so"))
    for cmd in ([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-Xcompiler", "-fPIC", *inc, "-c", os.path.join(src, "runtime.cu"), "-o", a],
                ["g++", "-O1", "-std=c++17", "-fPIC", *inc, "-I", os.path.join(cuda, "include"), "-c", os.path.join(ROOT, "tests", "fake_cuda", "standin.cpp"), "-o", b],
                ["g++", "-shared", "-Wl,-Bsymbolic", "-Wl,-z,defs", a, b, "-o", out]):
        res = subprocess.run(cmd, capture_output=True, text=True)
        assert res.returncode == 0, res.stderr
    lib = ctypes.CDLL(out)
    for name, (res, args) in _lib.SIGNATURES.items():
        if hasattr(lib, name):
            getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    return lib


@pytest.fixture(scope="session")
def standin(tmp_path_factory):
    before = os.environ.get("DEEPJ_CUDA_NO_GRAPH")
    os.environ["DEEPJ_CUDA_NO_GRAPH"] = "1"
    try:
        lib = build(str(tmp_path_factory.mktemp("standin")))
        assert lib.deepj_cuda_init(0) == 0
    finally:
        if before is None:
            del os.environ["DEEPJ_CUDA_NO_GRAPH"]
        else:
            os.environ["DEEPJ_CUDA_NO_GRAPH"] = before
    return lib


@pytest.fixture
def box(standin, monkeypatch):
    """The package on the stand-in, with nothing allocated."""
    monkeypatch.setattr(_lib, "_lib", standin)
    b = Box(standin)
    yield b
    b.close()


class Box:
    _next = 1 << 20

    def __init__(self, lib):
        self.lib, self.ids, self.rt = lib, [], cg.CudaGpuRuntime()
        self.launched()

    def id(self):
        Box._next += 1
        self.ids.append(Box._next)
        return Box._next

    def buf(self, data):
        a, i = np.ascontiguousarray(data, dtype=np.float32), self.id()
        self.rt.alloc_buffers([i], [a.size], 1)
        if a.size:
            self.rt.upload_buffer(i, a)
        return i

    def zeros(self, n):
        i = self.id()
        self.rt.alloc_buffers([i], [n], 1)
        return i

    def get(self, i, n):
        out = np.empty(n, dtype=np.float32)
        self.rt.download_buffer(i, out)
        return out

    def cache(self, layers, B, G, S, hd):
        i = self.id()
        _lib.check(self.lib.deepj_cuda_kv_alloc_q4(i, layers, B, G, S, hd))
        return i

    def flush(self, *words):
        s = cg.stream(words)
        self.rt.flush_ops(s, s.size)

    def launched(self):
        """(kind, three numbers) of every launch since the last call."""
        out = (ctypes.c_int * (4 * 4096))()
        n = self.lib.standin_notes(out, 4096)
        return [tuple(out[4 * i:4 * i + 4]) for i in range(n)]

    def close(self):
        self.rt.release_buffers(self.ids, len(self.ids))
