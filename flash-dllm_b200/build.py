"""Build ``libflashdllm_b200.so`` (the C-ABI library) in-tree with nvcc.

    python -m flash_dllm_b200.build          # or: python flash-dllm_b200/build.py

Every ``csrc/*.cu`` is compiled for sm_100a only (``-gencode
arch=compute_100a,code=sm_100a -lineinfo -O3``) into ``_build/`` at the repo
root and linked into ``flash-dllm_b200/libflashdllm_b200.so`` next to this
file.  ``csrc/torch_ops.cpp`` (the torch binding of the quantised operators)
is compiled with g++ against the installed torch and linked to that library
as ``_torch_ops.so``.  Objects are rebuilt when a source or header is newer,
the binding also when another torch or Python or other flags built it.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(ROOT, "_build")
LIB = os.path.join(PKG, "libflashdllm_b200.so")
BINDING_SRC = os.path.join(CSRC, "torch_ops.cpp")
BINDING = os.path.join(PKG, "_torch_ops.so")
BINDING_STAMP = os.path.join(BUILD, "_torch_ops.stamp")  # what the binding was built with
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-I", INCLUDE,
         "-I", CSRC]


def _nvcc() -> str:
    for c in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found (needed to build the sm_100a library)")


def _newest_dep() -> float:
    deps = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + \
        glob.glob(os.path.join(INCLUDE, "*.h"))
    return max(os.path.getmtime(d) for d in deps) if deps else 0.0


def _binding_cmd() -> list:
    from torch.utils import cpp_extension as ext
    inc = [*ext.include_paths("cuda"), sysconfig.get_paths()["include"], INCLUDE]
    libs = ext.library_paths("cuda")
    # (the system's g++: the module has to share torch's libstdc++, which a
    # compiler that links its own statically would not)
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            "-DTORCH_EXTENSION_NAME=_torch_ops", *[f"-I{p}" for p in inc], BINDING_SRC, "-o", BINDING,
            *[f"-L{p}" for p in libs], "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-lc10", "-lc10_cuda",
            f"-L{PKG}", f"-l:{os.path.basename(LIB)}", "-Wl,-rpath,$ORIGIN"]


def _binding_stamp(cmd: list) -> str:
    import torch
    return "\n".join([sys.version, torch.__version__, str(torch.version.git_version), *cmd])


def _binding_stale(stamp: str, dep_t: float) -> bool:
    """Whether the binding is missing, older than its source or a header, or
    built for another torch (its C++ interface is not stable), Python or path."""
    if not os.path.exists(BINDING) or os.path.getmtime(BINDING) < max(os.path.getmtime(BINDING_SRC), dep_t):
        return True
    try:
        with open(BINDING_STAMP) as f:
            return f.read() != stamp
    except FileNotFoundError:
        return True


def build(verbose: bool = False, force: bool = False) -> str:
    nvcc = _nvcc()
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    dep_t = _newest_dep()
    jobs = []
    objs = []
    for s in srcs:
        o = os.path.join(BUILD, os.path.basename(s)[:-3] + ".o")
        objs.append(o)
        if force or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), dep_t):
            jobs.append([nvcc, *ARCH, *FLAGS, "-c", s, "-o", o])

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
        if verbose and (r.stdout or r.stderr):
            print(r.stdout, r.stderr, file=sys.stderr)

    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        list(ex.map(run, jobs))
    if jobs or not os.path.exists(LIB) or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs):
        run([nvcc, *ARCH, "-shared", "-o", LIB, *objs, "-lcudart_static", "-lrt", "-ldl", "-lpthread"])
    cmd = _binding_cmd()
    stamp = _binding_stamp(cmd)
    if force or _binding_stale(stamp, dep_t):
        run(cmd)
        with open(BINDING_STAMP, "w") as f:
            f.write(stamp)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
