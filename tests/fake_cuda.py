"""The library's host code on a stand-in CUDA runtime (fake_cudart.cpp): what it
would launch, allocate and order, without a GPU."""
import ctypes
import pathlib
import shutil
import subprocess
import sys

import pytest

import sgblas_b200 as sg

ROOT = pathlib.Path(__file__).resolve().parent.parent
OBJECTS = ROOT / "sgblas_b200" / "_build"
CUDA = "/usr/local/cuda"
FAKE = 0x10000   # an address that nothing reads, 64 KiB aligned


def build(folder: pathlib.Path) -> ctypes.CDLL:
    """The library's objects linked with the stand-in, as a library of its own."""
    if shutil.which("g++") is None or not pathlib.Path(CUDA, "include", "cuda.h").exists():
        pytest.skip("g++ and the CUDA headers are needed")
    # Compiles what is out of date, which is nothing after a build.
    subprocess.run([sys.executable, str(ROOT / "sgblas_b200" / "build.py")], check=True,
                   capture_output=True)
    objects = sorted(str(OBJECTS / (p.name + ".o")) for p in (ROOT / "sgblas_b200" / "csrc").iterdir()
                     if p.suffix in (".cu", ".cpp"))
    so = folder / "libsgblas_fake.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CUDA}/include",
                    str(ROOT / "tests" / "fake_cudart.cpp"), *objects, "-o", str(so), "-Wl,-Bsymbolic",
                    "-Wl,--no-undefined", "-ldl", "-lpthread", "-lrt"], check=True)
    dll = ctypes.CDLL(str(so))
    for name, (res, args) in sg._SIGNATURES.items():
        fn = getattr(dll, name)
        fn.restype, fn.argtypes = res, args
    dll.fakeLog.restype = dll.fakeKernels.restype = ctypes.c_char_p
    return dll


def demangled(names):
    text = subprocess.run(["c++filt"], input="\n".join(names), text=True, capture_output=True,
                          check=True).stdout
    for scope in ("sgblas::kern::prod::", "sgblas::detail::"):
        text = text.replace(scope, "")
    return text.splitlines()


class Log:
    """What the library did since the last reset."""

    def __init__(self, dll):
        self.dll = dll

    def lines(self):
        return self.dll.fakeLog().decode().splitlines()

    def launches(self):
        """(kernel, grid.x) of each launch, kernels as their demangled names."""
        found = [line.split()[1:] for line in self.lines() if line.startswith("launch ")]
        return list(zip(demangled(f[0] for f in found), (int(f[1]) for f in found)))

    def shapes(self):
        """(kernel, grid.x, block.x, block.y, dynamic shared memory) of each launch."""
        found = [line.split()[1:] for line in self.lines() if line.startswith("launch ")]
        return [(name, *map(int, f[1:])) for name, f in zip(demangled(f[0] for f in found), found)]

    def kernels(self):
        """Every kernel that the library has."""
        return set(demangled(self.dll.fakeKernels().decode().split()))
