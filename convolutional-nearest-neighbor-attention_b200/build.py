"""Build libconvnn_b200.so in-tree with nvcc for sm_100a (no other architecture).

    python convolutional-nearest-neighbor-attention_b200/build.py [--force] [-v]

Each .cu under csrc/ is compiled to an object file (in parallel) and the objects are
linked into one shared library next to this file.  A source is recompiled when it, any
header under csrc/ or include/, or this script is newer than its object.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import threading
import warnings
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libconvnn_b200.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
CFLAGS = ARCH + ["-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-Xptxas", "-v", "-I", INCLUDE]


def sources() -> list:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _headers() -> list:
    return glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h")) + [os.path.abspath(__file__)]


def _obj(src: str) -> str:
    return os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")


def _newer(path: str, than: float) -> bool:
    return os.path.getmtime(path) > than


STAMP = LIB + ".srchash"


def source_hash() -> str:
    """Digest of every file the library is built from (content, not timestamps, so a copy
    of the tree with a prebuilt library is not rebuilt)."""
    import hashlib
    h = hashlib.sha256()
    for f in sorted(sources() + _headers()):
        h.update(os.path.basename(f).encode())
        with open(f, "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()


def stale() -> bool:
    if not os.path.exists(LIB) or not os.path.exists(STAMP):
        return True
    with open(STAMP) as f:
        return f.read().strip() != source_hash()


# The host side of some calls as a Python extension module, against the headers of the torch that is installed.
CALL_SRC = os.path.join(CSRC, "fp8_call.cpp")
CALL_LIB = os.path.join(HERE, "_fp8_call.so")
CALL_STAMP = CALL_LIB + ".srchash"


def call_hash() -> str:
    """Digest of the module's source, of the library's header, whose signatures it calls, and of what else its binary
    depends on."""
    import hashlib
    import torch
    h = hashlib.sha256(f"{sys.version_info[:2]} {torch.__version__}".encode())
    for name in (CALL_SRC, os.path.join(INCLUDE, "convnn_b200.h")):
        with open(name, "rb") as f:
            h.update(f.read())
    return h.hexdigest()


def call_stale() -> bool:
    if not os.path.exists(CALL_LIB) or not os.path.exists(CALL_STAMP):
        return True
    with open(CALL_STAMP) as f:
        return f.read().strip() != call_hash()


def build_call() -> str:
    import sysconfig
    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
               os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++20", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    tmp = f"{CALL_LIB}.{os.getpid()}.{threading.get_ident()}.tmp"        # (ranks and threads may build at the same time)
    cmd += [f"-isystem{i}" for i in include] + ["-I" + INCLUDE, CALL_SRC, "-o", tmp, "-L" + os.path.join(root, "lib")]
    cmd += ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"g++ failed on {os.path.basename(CALL_SRC)}:\n{r.stderr[-8000:]}")
        os.replace(tmp, CALL_LIB)
        with open(tmp, "w") as f:
            f.write(call_hash())
        os.replace(tmp, CALL_STAMP)
    finally:
        if os.path.exists(tmp):
            os.remove(tmp)
    return CALL_LIB


def _nvcc() -> str:
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found: the CUDA library cannot be built")
    return nvcc


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile what changed and link; return the library's path.  The host side of some calls is built after it; without
    that module the calls go through Python."""
    path = build_library(force, verbose)
    try:
        if force or call_stale():
            build_call()
    except (RuntimeError, ImportError, OSError) as e:        # the compiler, torch, a folder
        warnings.warn(f"the host side of the 8-bit calls is not built, they go through Python: {e}", RuntimeWarning)
    return path


def build_library(force: bool = False, verbose: bool = False) -> str:
    if not force and not stale():
        return LIB
    nvcc = _nvcc()
    os.makedirs(OBJ, exist_ok=True)
    hdr_t = max(os.path.getmtime(h) for h in _headers())
    todo = []
    for s in sources():
        o = _obj(s)
        if force or not os.path.exists(o) or _newer(s, os.path.getmtime(o)) or hdr_t > os.path.getmtime(o):
            todo.append(s)

    def compile_one(s: str):
        cmd = [nvcc] + CFLAGS + ["-c", s, "-o", _obj(s)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        return s, r.returncode, " ".join(cmd) + "\n" + r.stdout + r.stderr

    logs = []
    with ThreadPoolExecutor(max_workers=min(8, max(1, len(todo)))) as ex:
        for s, rc, log in ex.map(compile_one, todo):
            logs.append(log)
            if rc != 0:
                raise RuntimeError(f"nvcc failed on {os.path.basename(s)}:\n{log[-8000:]}")
    cmd = [nvcc] + ARCH + ["-shared", "-cudart", "static", "-o", LIB + ".tmp"] + [_obj(s) for s in sources()]
    r = subprocess.run(cmd, capture_output=True, text=True)
    logs.append(" ".join(cmd) + "\n" + r.stdout + r.stderr)
    with open(os.path.join(OBJ, "build.log"), "a" if not force else "w") as f:
        f.write("\n".join(logs))
    if r.returncode != 0:
        raise RuntimeError("link failed:\n" + logs[-1][-8000:])
    os.replace(LIB + ".tmp", LIB)
    with open(STAMP, "w") as f:
        f.write(source_hash())
    if verbose:
        print("\n".join(logs))
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
