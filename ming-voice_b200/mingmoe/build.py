"""Build the C-ABI library `libmingmoe.so` from `csrc/*.cu` with nvcc, in-tree, for sm_100a only.

    python ming-voice_b200/mingmoe/build.py [-v] [--force]

Each translation unit compiles to an object under `mingmoe/_build/` (skipped when up to date), then they
link into `mingmoe/libmingmoe.so` next to this file. The CUDA runtime is linked statically, so the library
depends only on the driver. `csrc/attention_host.cpp`, the host side of the attention calls, becomes the Python module
`mingmoe/_attention_host.so` beside it (g++, torch's headers; no device code).
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
CSRC = os.path.join(PKG, "csrc")
ROOT = os.path.dirname(PKG)
INCLUDE = os.path.join(ROOT, "include")
OUT = os.path.join(HERE, "libmingmoe.so")
BUILD = os.path.join(HERE, "_build")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-Xcompiler", "-fvisibility=hidden", "-I", CSRC, "-I", INCLUDE]


def nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def _deps():
    return sorted(glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) +
                  glob.glob(os.path.join(INCLUDE, "*.h")))


def _compile(src: str, verbose: bool, ptxas_v: bool, build_dir: str = BUILD, extra=()) -> str:
    obj = os.path.join(build_dir, os.path.basename(src) + ".o")
    newest_dep = max([os.path.getmtime(src)] + [os.path.getmtime(d) for d in _deps()])
    if os.path.exists(obj) and os.path.getmtime(obj) >= newest_dep and not ptxas_v:
        return obj
    cmd = [nvcc(), *ARCH, *FLAGS, *extra, "-c", src, "-o", obj]
    if ptxas_v:
        cmd += ["-Xptxas", "-v"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    if ptxas_v or verbose:
        sys.stdout.write(r.stderr)
    return obj


def build(verbose: bool = False, force: bool = False, ptxas_v: bool = False, out: str = OUT, build_dir: str = BUILD,
          extra=()) -> str:
    """Compile and link; `out`, `build_dir` and `extra` nvcc flags select a variant build (e.g. -DMV_TRACE for
    the phase-timing stamps of the decode kernel) without touching the default library."""
    OUT = out
    os.makedirs(build_dir, exist_ok=True)
    if force:
        for f in glob.glob(os.path.join(build_dir, "*.o")):
            os.remove(f)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose, ptxas_v, build_dir, tuple(extra)), srcs))
    if (not os.path.exists(OUT) or force or ptxas_v or
            max(os.path.getmtime(o) for o in objs) > os.path.getmtime(OUT)):
        tmp = OUT + ".tmp"
        cmd = [nvcc(), *ARCH, "-shared", "-o", tmp, *objs, "-cudart", "static"]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, OUT)
    return OUT


HOST_SRC = os.path.join(CSRC, "attention_host.cpp")
HOST_OUT = os.path.join(HERE, "_attention_host.so")


def build_host(verbose: bool = False, force: bool = False) -> str:
    """The Python module `_attention_host`. It is bound to the headers of one torch and one Python, so the command that compiled
    it (with their versions) is kept beside the objects, and another command compiles it again."""
    import sysconfig

    import torch
    tdir = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    inc = [os.path.join(tdir, "include"), os.path.join(tdir, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(cuda, "include"), INCLUDE]
    tmp = HOST_OUT + ".tmp"
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{d}" for d in inc], HOST_SRC, "-o",
           tmp, f"-L{os.path.join(tdir, 'lib')}", "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10"]
    made_by = f"torch {torch.__version__}, python {sys.version}: {' '.join(cmd).replace(ROOT, '.')}\n"
    record = os.path.join(BUILD, "attention_host.cmd")
    newest = max([os.path.getmtime(p) for p in [HOST_SRC, *glob.glob(os.path.join(INCLUDE, "*.h"))]])
    if os.path.exists(HOST_OUT) and os.path.getmtime(HOST_OUT) >= newest and not force and os.path.exists(record):
        with open(record) as f:
            if f.read() == made_by:
                return HOST_OUT
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {HOST_SRC}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, HOST_OUT)
    os.makedirs(BUILD, exist_ok=True)
    with open(record, "w") as f:
        f.write(made_by)
    return HOST_OUT


if __name__ == "__main__":
    print(build_host(verbose="-v" in sys.argv, force="--force" in sys.argv))
    print(build(verbose="-v" in sys.argv, force="--force" in sys.argv, ptxas_v="--ptxas" in sys.argv))
