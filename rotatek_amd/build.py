"""Build librotatek_hip.so in-tree with hipcc for gfx950.

``python -m rotatek_amd.build`` (or ``__graft_entry__.build()``) compiles
every ``csrc/*.hip`` translation unit in parallel and links them into
``rotatek_amd/librotatek_hip.so``.  All HIP code is compiled with packed
fp32 instructions disabled (``-target-feature -packed-fp32-ops``).  Beside
it ``rotatek_amd/_bind.so``, host code alone: ``csrc/rk_bind.cpp`` against
torch's headers.
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
INCLUDE = os.path.join(ROOT, "include")
LIB_NAME = "librotatek_hip.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
BIND_PATH = os.path.join(HERE, "_bind.so")
ARCH = os.environ.get("ROTATEK_OFFLOAD_ARCH", "gfx950")

COMMON_FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", f"-I{INCLUDE}", f"-I{CSRC}",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (ROCm is required to build the HIP library)")


def _compile(hipcc: str, src: str, obj: str, verbose: bool) -> None:
    cmd = [hipcc, *COMMON_FLAGS, "-c", src, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed on {os.path.basename(src)}:\n{res.stderr[-4000:]}")


def _build_bind(hipcc: str, verbose: bool) -> None:
    """The Python module of host code (torch only when it is built)."""
    import torch
    cxx = shutil.which("g++") or shutil.which("c++") or hipcc
    inc, lib = (os.path.join(os.path.dirname(torch.__file__), d) for d in ("include", "lib"))
    tmp = BIND_PATH + ".tmp"
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
           "-isystem", sysconfig.get_paths()["include"], "-isystem", inc,
           "-isystem", os.path.join(inc, "torch", "csrc", "api", "include"),
           os.path.join(CSRC, "rk_bind.cpp"), "-o", tmp, f"-L{lib}", "-ltorch_python", "-ltorch_cpu", "-lc10"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cxx)} failed on rk_bind.cpp:\n{res.stderr[-4000:]}")
    os.replace(tmp, BIND_PATH)


def build(verbose: bool = False, jobs: int | None = None) -> str:
    """Compile and link the library; returns its path."""
    hipcc = _hipcc()
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    objs = [os.path.join(objdir, os.path.basename(s)[:-4] + ".o") for s in srcs]
    jobs = jobs or min(len(srcs), max(1, (os.cpu_count() or 4)))
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        futs = [ex.submit(_build_bind, hipcc, verbose)]
        futs += [ex.submit(_compile, hipcc, s, o, verbose) for s, o in zip(srcs, objs)]
        for f in futs:
            f.result()
    tmp = LIB_PATH + ".tmp"
    cmd = [hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr[-4000:]}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
