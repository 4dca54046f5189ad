"""Build libssa_sm100a.so in-tree with nvcc (sm_100a only).

    python -m ssa_b200.build [--verbose]

Every ``csrc/*.cu`` file is compiled for ``-gencode arch=compute_100a,code=sm_100a``
and linked into ``ssa_b200/libssa_sm100a.so`` (CUDA runtime linked statically).
``csrc/paged_call.cpp``, the argument path of the paged-cache ops from Python, becomes
the extension module ``ssa_b200/_paged_call.so`` (it uses PyTorch's C++ headers and
calls the library; the library itself depends on neither).
The shared object sits next to this file so that it travels with the source
tree; it is rebuilt only when a source or header is newer than it.
"""

from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libssa_sm100a.so")
BUILD = os.path.join(ROOT, "_build")
CALL_SRC = os.path.join(CSRC, "paged_call.cpp")
CALL_LIB = os.path.join(HERE, "_paged_call.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
              "-Xptxas", "-warn-spills", "-I" + os.path.join(ROOT, "include")]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found: the sm_100a library cannot be built")
    return cand


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def build_call(force: bool = False) -> str:
    """Compile the extension module (a host compiler, no CUDA); return its path."""
    deps = [CALL_SRC, os.path.join(ROOT, "include", "ssa_b200.h")]
    if not force and os.path.exists(CALL_LIB) and all(os.path.getmtime(f) <= os.path.getmtime(CALL_LIB) for f in deps):
        return CALL_LIB
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    cxx = shutil.which("g++") or "g++"
    inc = [f"-isystem{d}" for d in include_paths() + [sysconfig.get_paths()["include"], "/usr/local/cuda/include"]]
    libs = [f"-L{d}" for d in library_paths()] + ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    tmp = CALL_LIB + ".tmp"
    cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *inc, CALL_SRC, "-o", tmp, *libs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cxx} failed on {CALL_SRC}:\n{r.stderr[-4000:]}")
    os.replace(tmp, CALL_LIB)
    return CALL_LIB


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(ROOT, "include", "*.h"))
    return any(os.path.getmtime(f) > t for f in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile and link the library and the extension module; return the library's path."""
    if not force and not _stale():
        build_call()
        return LIB
    nvcc = _nvcc()
    os.makedirs(BUILD, exist_ok=True)
    extra = ["-Xptxas", "-v"] if verbose else []

    def compile_one(src):
        obj = os.path.join(BUILD, os.path.basename(src) + ".o")
        cmd = [nvcc, *ARCH, *NVCC_FLAGS, *extra, "-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{r.stderr}")
        return obj, r.stderr

    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        call = ex.submit(build_call, force)
        results = list(ex.map(compile_one, sources()))
    call.result()
    if verbose:
        for _, log in results:
            sys.stderr.write(log)
    objs = [o for o, _ in results]
    tmp = LIB + ".tmp"
    cmd = [nvcc, *ARCH, "-shared", "-cudart", "static", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose="--verbose" in sys.argv))
