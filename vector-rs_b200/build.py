"""Builds libvrs.so (the sm_100a CUDA library behind include/vrs.h) in-tree.

    python vector-rs_b200/build.py [--force] [-v]

Each csrc/*.cu is compiled by nvcc for sm_100a only into _build/, then
linked with the static CUDA runtime and NCCL into lib/libvrs.so. Where a torch
with CUDA is installed, csrc/py_ops.cpp becomes python/vector_cuda/_ops.so,
again whenever that torch changes. The
generator (gen_kernels.cu) is compiled without FMA contraction on both the
device and the host so its output is bit-identical everywhere.
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(PKG, "_build")
LIBDIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIBDIR, "libvrs.so")
# The torch side of vector_cuda.ops.
OPS_SRC = os.path.join(CSRC, "py_ops.cpp")
OPS = os.path.join(PKG, "python", "vector_cuda", "_ops.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr",
          "-Xcompiler", "-fPIC,-ffp-contract=off,-fvisibility=hidden",
          "-I", os.path.join(ROOT, "include")]
PER_FILE = {"gen_kernels.cu": ["-fmad=false"]}


def nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def sources() -> list[str]:
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers_mtime() -> float:
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs.append(os.path.join(ROOT, "include", "vrs.h"))
    return max(os.path.getmtime(h) for h in hs)


def _compile(src: str, force: bool, verbose: bool) -> str:
    obj = os.path.join(BUILD, src.replace(".cu", ".o"))
    path = os.path.join(CSRC, src)
    if (not force and os.path.exists(obj)
            and os.path.getmtime(obj) >= max(os.path.getmtime(path), _headers_mtime())):
        return obj
    cmd = [nvcc(), *ARCH, *COMMON, *PER_FILE.get(src, []), "-c", path, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
    if verbose and r.stderr.strip():
        print(r.stderr, flush=True)
    return obj


def _ops_stamp(torch: str) -> str:
    """What _ops.so is built against: the torch, by place and version, and the Python."""
    try:
        with open(os.path.join(torch, "version.py")) as f:
            version = f.read()
    except OSError:
        version = ""
    return "\n".join((torch, sys.version, version))


def build_ops(force: bool = False, verbose: bool = False) -> str | None:
    """_ops.so against the installed torch's headers; None, with a line that says
    so, where there is no torch with CUDA or no Python headers."""
    spec = importlib.util.find_spec("torch")
    torch = list(spec.submodule_search_locations)[0] if spec and spec.submodule_search_locations else None
    python = sysconfig.get_paths()["include"]
    lacks = ("torch" if torch is None else
             "a torch with CUDA" if not os.path.exists(os.path.join(torch, "lib", "libc10_cuda.so")) else
             "Python's headers" if not os.path.exists(os.path.join(python, "Python.h")) else None)
    if lacks:
        print(f"vector_cuda.ops is not built: it needs {lacks}", file=sys.stderr, flush=True)
        return None
    header = os.path.join(ROOT, "include", "vrs.h")
    stamp, want = os.path.join(BUILD, "ops.stamp"), _ops_stamp(torch)
    if (not force and os.path.exists(OPS) and os.path.exists(stamp)
            and os.path.getmtime(OPS) >= max(os.path.getmtime(OPS_SRC), os.path.getmtime(header))):
        with open(stamp) as f:
            if f.read() == want:
                return OPS
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    inc = [os.path.join(ROOT, "include"), os.path.join(torch, "include"),
           os.path.join(torch, "include", "torch", "csrc", "api", "include"),
           os.path.join(cuda, "include"), python]
    cmd = ["g++", "-O2", "-std=c++20", "-fPIC", "-shared", "-fvisibility=hidden", *[f"-isystem{i}" for i in inc],
           OPS_SRC, "-o", OPS, "-L" + os.path.join(torch, "lib"), "-Wl,-rpath," + os.path.join(torch, "lib"),
           "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on py_ops.cpp:\n{r.stdout}\n{r.stderr}")
    with open(stamp, "w") as f:
        f.write(want)
    return OPS


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    with ThreadPoolExecutor(max_workers=os.cpu_count() or 4) as ex:
        ops = ex.submit(build_ops, force, verbose)
        objs = list(ex.map(lambda s: _compile(s, force, verbose), sources()))
    newest = max(os.path.getmtime(o) for o in objs)
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < newest:
        cmd = [nvcc(), *ARCH, "-shared", "-o", LIB, *objs, "-cudart", "static", "-lnccl"]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    ops.result()  # last: the library does not need the extension
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    args = ap.parse_args()
    print(build(args.force, args.verbose))
    sys.exit(0)
