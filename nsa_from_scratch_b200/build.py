"""Builds libnsa_b200.so (the C-ABI library) in-tree with nvcc for sm_100a, and _nsa_torch.so beside it: the layer's
operators on torch tensors, host code over that library (csrc/torch_ops.cpp, compiled for the torch at hand).

    python -m nsa_from_scratch_b200.build [--force] [--verbose]

Each .cu under csrc/ is compiled to an object file (in parallel) and the objects are
linked into nsa_from_scratch_b200/libnsa_b200.so.  A stamp of the source hashes makes
repeated calls free.  nvcc cross-compiles, so no GPU is needed to build.
"""
from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libnsa_b200.so")
INC = os.path.join(os.path.dirname(PKG), "include")
TORCH_LIB = os.path.join(PKG, "_nsa_torch.so")
TORCH_SRC = os.path.join(CSRC, "torch_ops.cpp")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-Xptxas", "-v",
]


class NoCompiler(RuntimeError):
    """This machine has no nvcc: what was built elsewhere may be used as it is."""


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise NoCompiler("nvcc not found; set NVCC")


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _digest() -> str:
    h = hashlib.sha256()
    for root in (CSRC, INC):
        for f in sorted(os.listdir(root)):
            if f.endswith((".cu", ".cuh", ".h")):
                h.update(f.encode())
                h.update(open(os.path.join(root, f), "rb").read())
    h.update(" ".join(NVCC_FLAGS).encode())
    return h.hexdigest()


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile if sources changed; return the path of the shared library."""
    stamp = os.path.join(OBJ, "stamp")
    dig = _digest()
    if not force and os.path.exists(LIB) and os.path.exists(stamp) and open(stamp).read() == dig:
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    nvcc = _nvcc()

    def one(src):
        obj = os.path.join(OBJ, src[:-3] + ".o")
        cmd = [nvcc, *NVCC_FLAGS, "-I", INC, "-c", os.path.join(CSRC, src), "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        with open(os.path.join(OBJ, src[:-3] + ".ptxas.log"), "w") as f:
            f.write(r.stderr)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{r.stderr[-4000:]}")
        if verbose:
            print(r.stderr)
        return obj

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(one, _sources()))
    r = subprocess.run([nvcc, "-shared", "-o", LIB, *objs, "-lcudart"], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr[-4000:]}")
    with open(stamp, "w") as f:
        f.write(dig)
    return LIB


def build_torch(force: bool = False) -> str:
    """Compile the torch side if its source, the C header, torch or Python changed; return the path of the module."""
    import sysconfig

    import torch

    build()
    h = hashlib.sha256(f"{torch.__version__} {torch._C._GLIBCXX_USE_CXX11_ABI} {sys.version}".encode())
    for f in (TORCH_SRC, os.path.join(INC, "nsa_b200.h"), os.path.abspath(__file__)):
        h.update(open(f, "rb").read())
    stamp, dig = os.path.join(OBJ, "torch_stamp"), h.hexdigest()
    if not force and os.path.exists(TORCH_LIB) and os.path.exists(stamp) and open(stamp).read() == dig:
        return TORCH_LIB
    # nvcc's host compiler, as for the library.  $CXX may be another one that links a C++ runtime of its own into the module,
    # and with two of them in one process the first formatted error message crashes.
    nvcc = _nvcc()
    home, cuda = os.path.dirname(torch.__file__), os.path.dirname(os.path.dirname(os.path.realpath(nvcc)))
    part = f"{TORCH_LIB}.{os.getpid()}"              # renamed when whole: two processes may build at once
    cmd = [nvcc, "-O2", "-std=c++17", "-shared", "-cudart", "none", "-Xcompiler", "-fPIC,-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_nsa_torch",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-I{d}" for d in (os.path.join(home, "include"), os.path.join(home, "include/torch/csrc/api/include"), os.path.join(cuda, "include"),
                                sysconfig.get_paths()["include"])),
           TORCH_SRC, "-o", part, f"-L{home}/lib", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python", f"-L{PKG}",
           "-Xlinker", "-l:libnsa_b200.so", "-Xlinker", "-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on torch_ops.cpp:\n{r.stderr[-4000:]}")
    os.replace(part, TORCH_LIB)
    with open(stamp, "w") as f:
        f.write(dig)
    return TORCH_LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
    print(build_torch(force="--force" in sys.argv))
