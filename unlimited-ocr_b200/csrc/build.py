"""Build libsrswa.so (sm_100a) in-tree with nvcc.

    python unlimited-ocr_b200/csrc/build.py [--force]

Objects are compiled in parallel into ``unlimited-ocr_b200/csrc/_build/`` and
linked into ``unlimited-ocr_b200/srswa/libsrswa.so``.  The CUDA runtime is linked
statically, so the library only needs the NVIDIA driver at run time (and loads,
without a GPU, on a build host).  ``srswa/_bind.so`` is the Python binding of the
entries that a decode step calls once per layer; it needs a C++ compiler and the
headers of the installed torch (with CUDA).  Where they are missing the library is
built without it, and those calls raise.
"""

from __future__ import annotations

import concurrent.futures as cf
import importlib.metadata
import importlib.util
import os
import shutil
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


def _bind(force: bool) -> str:
    """Builds the binding if it is older than its sources or made for another
    torch or interpreter.  Returns why it cannot be built here ("": it is
    there)."""
    spec = importlib.util.find_spec("torch")
    if spec is None:
        return "torch is not installed"
    torch = spec.submodule_search_locations[0]
    if not os.path.exists(os.path.join(torch, "include", "c10", "cuda", "CUDAStream.h")):
        return "the installed torch has no CUDA headers"
    src = os.path.join(HERE, "bind.cpp")
    deps = [src, os.path.join(ROOT, "include", "srswa.h")]
    key = "\n".join([importlib.metadata.version("torch"), torch, str(sysconfig.get_config_var("SOABI"))])
    mark = os.path.join(BUILD, "bind.key")
    made_for = open(mark).read() if os.path.exists(mark) else None
    if not force and made_for == key and os.path.exists(BIND) and all(os.path.getmtime(d) <= os.path.getmtime(BIND) for d in deps):
        return ""
    cxx = os.environ.get("CXX", "g++")
    if shutil.which(cxx) is None:
        return f"no C++ compiler ({cxx})"
    from torch import compiled_with_cxx11_abi
    cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(compiled_with_cxx11_abi())}", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(torch, "include"),
           "-I", os.path.join(torch, "include", "torch", "csrc", "api", "include"), "-I", sysconfig.get_paths()["include"],
           "-I", os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include"), src, "-o", BIND + ".tmp",
           "-L", os.path.join(torch, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-ldl"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"bind.cpp failed:\n{r.stdout}\n{r.stderr}")
    os.replace(BIND + ".tmp", BIND)
    with open(mark, "w") as f:
        f.write(key)
    return ""


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=min(8, len(SOURCES) + 1)) as ex:
        bind = ex.submit(_bind, force)
        objs = list(ex.map(lambda s: _compile(s, force, verbose), SOURCES))
    if force or not os.path.exists(OUT) or any(os.path.getmtime(o) > os.path.getmtime(OUT) for o in objs):
        cmd = [NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-cudart", "static",
               "-Xcompiler", "-fPIC", *objs, "-o", OUT + ".tmp"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(OUT + ".tmp", OUT)
    missing = bind.result()  # the library is there by now
    if missing:
        sys.stderr.write(f"_bind.so not built: {missing}; the scaled 8-bit cache's and the pages' calls need it\n")
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
