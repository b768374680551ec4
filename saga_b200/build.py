"""Build libsaga_b200.so (the C-ABI library) in-tree with nvcc for sm_100a.

    python -m saga_b200.build [--force]

Sources: saga_b200/csrc/*.cu. Output: saga_b200/libsaga_b200.so. The library
links the CUDA runtime statically and has no PyTorch dependency. The host calls
of the 4-bit cache operators (saga_b200/csrc/fastcall.cpp) are a CPython module
of their own, saga_b200/_fastcall.<ABI tag>.so, which knows torch and is bound to
the library at run time. It is built where torch is installed, and again after
a change of torch, Python or the compiler; callers of the C ABI alone do without.
"""
from __future__ import annotations

import argparse
import glob
import hashlib
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libsaga_b200.so")
STAMP = os.path.join(HERE, ".libsaga_b200.stamp")
FAST_SRC = os.path.join(CSRC, "fastcall.cpp")
FAST = os.path.join(HERE, "_fastcall" + sysconfig.get_config_var("EXT_SUFFIX"))

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
         "-Xcompiler", "-fvisibility=hidden", "-Xptxas", "-v"]
# SAGA_PHASE_TRACE=1 in the environment builds the diagnostic phase trace in
# (SagaAttnArgs.trace); the default build leaves it out of the kernels.
if os.environ.get("SAGA_PHASE_TRACE") == "1":
    FLAGS.append("-DSAGA_PHASE_TRACE=1")


def _nvcc() -> str:
    for c in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _digest() -> str:
    h = hashlib.sha256()
    files = _sources() + sorted(glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")))
    files += [FAST_SRC, os.path.join(REPO, "include", "saga_b200.h")]
    for f in files:
        with open(f, "rb") as fh:
            h.update(os.path.basename(f).encode())
            h.update(fh.read())
    h.update(" ".join(ARCH + FLAGS).encode())
    fast = _fast_command(FAST)
    if fast:  # what the call module takes from torch's headers and Python's depends on their versions
        import torch
        h.update(" ".join([*fast, torch.__version__, sys.version]).encode())
    return h.hexdigest()


def _stamped() -> str:
    """What the built files were made of, or nothing."""
    if not os.path.exists(STAMP):
        return ""
    with open(STAMP) as f:
        return f.read().strip()


def up_to_date() -> bool:
    if not os.path.exists(LIB) or (_fast_command(FAST) and not os.path.exists(FAST)):
        return False
    return _stamped() == _digest()


def _fast_command(out: str):
    """The g++ command of the torch-facing call module, or None without torch."""
    try:
        import torch
        from torch.utils.cpp_extension import include_paths, library_paths
    except ImportError:
        return None

    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", sysconfig.get_paths()["include"], "-I", os.path.join(os.path.dirname(_nvcc()), "..", "include")]
    for d in include_paths():
        cmd += ["-isystem", d]
    cmd += [FAST_SRC, "-o", out]
    for d in library_paths():
        cmd += ["-L", d]
    return cmd + ["-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python"]


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every .cu under csrc/ into libsaga_b200.so (objects in parallel)."""
    if not force and up_to_date():
        return LIB
    nvcc = _nvcc()
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    procs = []
    objs = []
    for src in _sources():
        obj = os.path.join(objdir, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        cmd = [nvcc, *ARCH, *FLAGS, "-I", os.path.join(REPO, "include"), "-dc" if False else "-c", src, "-o", obj]
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    fast_tmp = FAST + ".tmp"
    fast = _fast_command(fast_tmp)
    if fast:
        procs.append((FAST_SRC, subprocess.Popen(fast, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    else:
        print("torch is not installed: the library for the C ABI alone is built")
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if verbose or p.returncode:
            sys.stdout.write(out)
        if p.returncode:
            failed.append(src)
    if failed:
        raise RuntimeError(f"compiling failed for {failed}")
    tmp = LIB + ".tmp"
    cmd = [nvcc, *ARCH, "-shared", "-cudart", "static", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode:
        sys.stdout.write(r.stdout + r.stderr)
        raise RuntimeError("link failed")
    os.replace(tmp, LIB)
    if fast:
        os.replace(fast_tmp, FAST)
    with open(STAMP, "w") as f:
        f.write(_digest())
    return LIB


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))


if __name__ == "__main__":
    main()
