"""Build the native library ``ddq_b200/lib/libddq_b200.so`` in-tree.

Every ``csrc/*.cu`` file is compiled for sm_100a only
(``-gencode arch=compute_100a,code=sm_100a``) with relocatable device code
(but for WHOLE_PROGRAM), in parallel, then device-linked into one shared library
that exports the C ABI declared in ``include/ddq_b200.h``.  The library links the
CUDA runtime statically and does not depend on torch; a module beside it, host
code on torch's headers (``torch_path``), holds the tensor checks of the paged
operators.  Sources are rebuilt only when a ``.cu``/``.cuh``/header file is newer
than the library, or the module is not of this torch and Python.

    python -m ddq_b200.build            # build if stale
    python -m ddq_b200.build --force    # rebuild
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys
import warnings

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(REPO_DIR, "include")
BUILD_DIR = os.path.join(PKG_DIR, "_build")
LIB_DIR = os.path.join(PKG_DIR, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libddq_b200.so")
# the paged operators' checks and tensor handling as a CPython module on torch
TORCH_SRC = os.path.join(CSRC, "torch_paged.cpp")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-rdc=true", "-Xcompiler", "-fPIC",
              "-Xcompiler", "-O3", "--expt-relaxed-constexpr", "-I", INCLUDE]
# compiled without relocatable device code: a kernel that moves registers
# between its warpgroups (ptxas ignores that across compilation units).  Such a
# file refers to no device symbol of another one.
WHOLE_PROGRAM = ("paged_tc.cu",)


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the ddq_b200 CUDA library cannot be built")


def _sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps() -> list[str]:
    return (_sources() + glob.glob(os.path.join(CSRC, "*.cuh"))
            + glob.glob(os.path.join(INCLUDE, "*.h")) + [os.path.abspath(__file__)])


def is_stale() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    return any(os.path.getmtime(p) > t for p in _deps())


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(BUILD_DIR, os.path.basename(src)[:-3] + ".o")
    flags = NVCC_FLAGS
    if os.path.basename(src) in WHOLE_PROGRAM:
        flags = [f for f in NVCC_FLAGS if f != "-rdc=true"] + ["-DDDQ_WHOLE_PROGRAM"]
    cmd = [_nvcc(), *ARCH_FLAGS, *flags, "-c", src, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    if verbose and (r.stdout or r.stderr):
        sys.stderr.write(r.stdout + r.stderr)
    return obj


def torch_path() -> str:
    """Where the paged operators' module for this torch and this Python lies: it is
    compiled on torch's C++ classes and Python's C API, so a module of others is not
    a module for these."""
    import sysconfig

    import torch
    v = torch.version
    tag = f"{torch.__version__}-{v.cuda}-{str(v.git_version)[:8]}"
    tag += f"-cxx11abi{int(torch.compiled_with_cxx11_abi())}"
    return os.path.join(LIB_DIR, f"_paged-{tag}{sysconfig.get_config_var('EXT_SUFFIX')}")


def build_torch(force: bool = False) -> str:
    """The CPython module of the paged operators (host code only; it gets the
    library's entry points at run time)."""
    path = torch_path()
    deps = [TORCH_SRC, os.path.abspath(__file__)] + glob.glob(os.path.join(INCLUDE, "*.h"))
    if not force and os.path.exists(path) and \
            all(os.path.getmtime(path) >= os.path.getmtime(p) for p in deps):
        return path
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    os.makedirs(LIB_DIR, exist_ok=True)
    tmp = f"{path}.{os.getpid()}.tmp"
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
           "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           "-I", os.path.join(root, "include"),
           "-I", os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-I", sysconfig.get_paths()["include"], "-I", os.path.join(cuda, "include"), TORCH_SRC,
           "-L", os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch",
           "-ltorch_python", "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed for {TORCH_SRC}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, path)
    return path


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compile the library if needed; return its path."""
    if not force and not is_stale():
        return LIB_PATH
    os.makedirs(BUILD_DIR, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    srcs = _sources()
    with cf.ThreadPoolExecutor(max_workers=max(1, min(len(srcs), os.cpu_count() or 1))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    tmp = LIB_PATH + ".tmp"
    cmd = [_nvcc(), *ARCH_FLAGS, "-shared", "-rdc=true", "-Xcompiler", "-fPIC", *objs, "-o", tmp]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the library and the paged operators' module if needed; return the
    library's path.  The library needs neither Python's headers nor torch's: where
    the module does not build, that is a warning, and only ``ddq_b200.paged``
    raises (``build_torch`` does so itself)."""
    path = build_library(force, verbose)
    try:
        build_torch(force)
    except (RuntimeError, OSError) as e:
        warnings.warn(f"ddq_b200.paged is not available: {e}", RuntimeWarning, stacklevel=2)
    return path


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
