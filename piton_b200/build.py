"""Build libpiton_b200.so (all CUDA sources under csrc/) for sm_100a.

    python -m piton_b200.build            # incremental: recompiles changed sources only

Every ``csrc/*.cu`` file is compiled to an object under ``csrc/_build/`` with
``nvcc -gencode arch=compute_100a,code=sm_100a`` (in parallel), then linked
into ``piton_b200/libpiton_b200.so``.  nvcc cross-compiles, so this runs on a
machine without a GPU; the shared object travels with the source tree.
``csrc/decode_calls.cpp``, the argument marshalling of ``piton_b200.decode``, is
compiled against the installed torch into ``piton_b200/_decode_calls.so``; where that
cannot be done (no torch, no C++20 host compiler) the library is built all the same, with a
warning, and only ``piton_b200.decode`` is missing.
"""

from __future__ import annotations

import concurrent.futures as cf
import glob
import hashlib
import os
import shutil
import subprocess
import sys
import warnings

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(CSRC, "_build")
LIB = os.path.join(PKG, "libpiton_b200.so")
CALLS = os.path.join(PKG, "_decode_calls.so")
INCLUDE = os.path.join(REPO, "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
                     "--expt-relaxed-constexpr", "-I" + INCLUDE, "-I" + CSRC]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _digest(path: str, deps: list) -> str:
    h = hashlib.sha256()
    for p in [path] + deps:
        with open(p, "rb") as f:
            h.update(f.read())
    h.update(" ".join(NVCC_FLAGS).encode())
    return h.hexdigest()[:16]


def _compile(src: str, deps: list, verbose: bool) -> str:
    name = os.path.splitext(os.path.basename(src))[0]
    obj = os.path.join(OBJ, f"{name}.o")
    stamp = obj + ".sha"
    digest = _digest(src, deps)
    if os.path.exists(obj) and os.path.exists(stamp) and open(stamp).read() == digest:
        return obj
    cmd = [nvcc()] + NVCC_FLAGS + ["-c", src, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
    with open(stamp, "w") as f:
        f.write(digest)
    return obj


def _build_calls(verbose: bool) -> str:
    """The extension module of piton_b200.decode: host code only, built by g++."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    src, stamp = os.path.join(CSRC, "decode_calls.cpp"), os.path.join(OBJ, "decode_calls.sha")
    digest = _digest(src, [os.path.join(INCLUDE, "piton_b200.h")]) + torch.__version__
    if os.path.exists(CALLS) and os.path.exists(stamp) and open(stamp).read() == digest:
        return CALLS
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++20", "-shared", "-fPIC", "-fvisibility=hidden", src, "-o", CALLS,
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I" + INCLUDE,
           "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include"),
           *["-I" + p for p in include_paths()], *["-L" + p for p in library_paths()],
           "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-ltorch", "-lc10_cuda", "-lc10"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed on {src}:\n{r.stdout}\n{r.stderr}")
    with open(stamp, "w") as f:
        f.write(digest)
    return CALLS


def build(verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    headers = sorted(glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h")))
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        calls = ex.submit(_build_calls, verbose)
        objs = list(ex.map(lambda s: _compile(s, headers, verbose), sources))
    newest = max(os.path.getmtime(o) for o in objs)
    if not os.path.exists(LIB) or os.path.getmtime(LIB) < newest:
        cmd = [nvcc()] + ARCH + ["-shared", "-o", LIB] + objs + ["-lcuda"]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    try:
        calls.result()
    except Exception as e:
        if os.path.exists(CALLS):           # of an earlier build: it may not fit the library any more
            os.remove(CALLS)
        warnings.warn(f"{os.path.basename(CALLS)} was not built, piton_b200.decode cannot be used: {e}")
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
