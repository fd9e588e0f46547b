"""Build liblifb.so (the C-ABI CUDA library) in-tree for sm_100a.

    python -m hard_resets_compose_b200.build      # or build() from Python

nvcc compiles every csrc/*.cu for `-gencode arch=compute_100a,code=sm_100a`
and links them into hard_resets_compose_b200/lib/liblifb.so.  The build runs
on a machine without a GPU (nvcc cross-compiles); the .so travels with the
source tree to the GPU machine.  Rebuilds only when a source is newer.
"""
from __future__ import annotations

import concurrent.futures
import glob
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "liblifb.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
              "-Xcompiler", "-Wall", "-I", CSRC, "-I", INCLUDE]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: set NVCC or put CUDA's bin directory on PATH")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + \
        glob.glob(os.path.join(INCLUDE, "*.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False, defines=(), out: str = None) -> str:
    """Compile liblifb.so.  `defines` are extra -D flags (the build-time
    tunables of csrc/chunk_tma.cu); `out` builds to another path instead of
    the in-tree library."""
    target = out or LIB
    if out is None and not force and not _stale():
        return LIB
    libdir = os.path.dirname(target)
    os.makedirs(libdir, exist_ok=True)
    objdir = os.path.join(libdir, "obj" if out is None else "obj_" + os.path.basename(target))
    os.makedirs(objdir, exist_ok=True)
    nvcc = _nvcc()
    objs, cmds = [], []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src)[:-3] + ".o")
        cmds.append([nvcc, *ARCH, *NVCC_FLAGS, *[f"-D{d}" for d in defines], "-c", src, "-o", obj])
        objs.append(obj)
    # one nvcc per translation unit, as many at once as there are cores
    with concurrent.futures.ThreadPoolExecutor(max_workers=max(1, min(len(cmds), os.cpu_count() or 1))) as ex:
        for cmd, res in zip(cmds, ex.map(lambda c: subprocess.run(c, capture_output=True, text=True), cmds)):
            if verbose:
                print(" ".join(cmd))
            if res.stdout or res.stderr:
                print(res.stdout + res.stderr, end="", file=sys.stderr)
            if res.returncode:
                raise subprocess.CalledProcessError(res.returncode, cmd, res.stdout, res.stderr)
    tmp = target + ".tmp"
    cmd = [nvcc, *ARCH, "-shared", "-o", tmp, *objs, "-lcudart"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    os.replace(tmp, target)
    return target


# ---- the host binding of the sequence-model operators (csrc/host): torch's C++ autograd

BINDING_SRC = os.path.join(CSRC, "host", "seq_binding.cpp")


def binding_path() -> str:
    """Where the binding is built: one for each torch, whose C++ interface it uses."""
    import torch
    return os.path.join(LIBDIR, "lifb_seq-" + torch.__version__.replace("+", "_") + ".so")


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """Compile csrc/host/seq_binding.cpp (g++, about a minute) if it is missing or stale."""
    import sysconfig

    import torch
    target = binding_path()
    deps = [BINDING_SRC] + glob.glob(os.path.join(INCLUDE, "*.h"))
    if not force and os.path.exists(target) and all(os.path.getmtime(d) <= os.path.getmtime(target) for d in deps):
        return target
    gxx = os.environ.get("CXX") or shutil.which("g++")
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    if not gxx:
        raise RuntimeError("g++ not found: set CXX or put it on PATH")
    os.makedirs(LIBDIR, exist_ok=True)
    root = os.path.dirname(torch.__file__)
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(cuda, "include"), INCLUDE]
    tmp = f"{target}.{os.getpid()}.tmp"
    cmd = [gxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-DTORCH_EXTENSION_NAME=lifb_seq",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[x for d in inc for x in ("-isystem", d)],
           BINDING_SRC, "-o", tmp, "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch",
           "-ltorch_python"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    os.replace(tmp, target)
    return target


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
    print(build_binding(force="--force" in sys.argv, verbose=True))
