"""Build libsrswa.so (sm_100a) in-tree with nvcc.

    python unlimited-ocr_b200/csrc/build.py [--force]

Objects are compiled in parallel into ``unlimited-ocr_b200/csrc/_build/`` and
linked into ``unlimited-ocr_b200/srswa/libsrswa.so``.  The CUDA runtime is linked
statically, so the library only needs the NVIDIA driver at run time (and loads,
without a GPU, on a build host).  ``srswa/_bind.so`` is the Python binding of the
entries that a decode step calls once per layer; it needs the headers of the
installed torch.
"""

from __future__ import annotations

import concurrent.futures as cf
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
ROOT = os.path.dirname(PKG)
OUT = os.path.join(PKG, "srswa", "libsrswa.so")
BIND = os.path.join(PKG, "srswa", "_bind.so")
BUILD = os.path.join(HERE, "_build")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
SOURCES = ["api.cu", "route.cu", "attend.cu", "gather.cu", "gather_tc.cu", "page_gate.cu", "peer.cu", "kl.cu",
           "cache8.cu", "cache8_attend.cu", "cache8_prompt.cu", "pages.cu"]
FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "-I", os.path.join(ROOT, "include"), "-I", HERE,
    "--expt-relaxed-constexpr",
    "-DSRSWA_BUILD",
]


def _newer(src: str, dst: str) -> bool:
    if not os.path.exists(dst):
        return True
    t = os.path.getmtime(dst)
    deps = [src] + [os.path.join(HERE, f) for f in os.listdir(HERE) if f.endswith((".cuh", ".h"))]
    deps.append(os.path.join(ROOT, "include", "srswa.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src: str, force: bool, verbose: bool) -> str:
    obj = os.path.join(BUILD, os.path.splitext(src)[0] + ".o")
    path = os.path.join(HERE, src)
    if force or _newer(path, obj):
        cmd = [NVCC, *FLAGS, "-c", path, "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
        if verbose:
            sys.stderr.write(r.stderr)
    return obj


def _bind(force: bool) -> None:
    src = os.path.join(HERE, "bind.cpp")
    deps = [src, os.path.join(ROOT, "include", "srswa.h")]
    if not force and os.path.exists(BIND) and all(os.path.getmtime(d) <= os.path.getmtime(BIND) for d in deps):
        return
    torch = importlib.util.find_spec("torch").submodule_search_locations[0]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           "-D_GLIBCXX_USE_CXX11_ABI=1", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(torch, "include"),
           "-I", os.path.join(torch, "include", "torch", "csrc", "api", "include"), "-I", sysconfig.get_paths()["include"],
           "-I", os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include"), src, "-o", BIND + ".tmp",
           "-L", os.path.join(torch, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-ldl"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"bind.cpp failed:\n{r.stdout}\n{r.stderr}")
    os.replace(BIND + ".tmp", BIND)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=min(8, len(SOURCES) + 1)) as ex:
        bind = ex.submit(_bind, force)
        objs = list(ex.map(lambda s: _compile(s, force, verbose), SOURCES))
        bind.result()
    if force or not os.path.exists(OUT) or any(os.path.getmtime(o) > os.path.getmtime(OUT) for o in objs):
        cmd = [NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-cudart", "static",
               "-Xcompiler", "-fPIC", *objs, "-o", OUT + ".tmp"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(OUT + ".tmp", OUT)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
