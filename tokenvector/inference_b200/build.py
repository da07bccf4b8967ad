"""Build libtvq.so in-tree with nvcc for sm_100a (B200), and beside it
_tvq_torch.so, the decoding operators on torch tensors (csrc/tvq_torch.cpp).

The shared libraries land next to this file so that they travel with the
repository snapshot; nothing is installed into site-packages.  Objects are
compiled in parallel and rebuilt only when a source or header is newer,
_tvq_torch.so also when Python or torch is another one.  Without torch it is
left out: libtvq.so does not need it.
"""
from __future__ import annotations

import concurrent.futures as cf
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
OBJDIR = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libtvq.so")
TORCH_SRC = os.path.join(CSRC, "tvq_torch.cpp")
TORCH_LIB = os.path.join(HERE, "_tvq_torch.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-fvisibility=hidden",
                     "--expt-relaxed-constexpr", "-I", INCLUDE, "-I", CSRC]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return hs


def _compile(nvcc, src, obj, verbose):
    cmd = [nvcc] + NVCC_FLAGS + ["-c", src, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed for %s:\n%s%s" % (os.path.basename(src), r.stdout, r.stderr))
    return r.stderr


def _torch_stamp() -> str:
    """What _tvq_torch.so depends on beside its sources."""
    return "python %s, torch %s" % (sys.version, importlib.metadata.version("torch"))


def _build_torch(force: bool) -> None:
    """_tvq_torch.so: g++ against torch's headers, linked to libtvq.so beside it."""
    if importlib.util.find_spec("torch") is None:
        sys.stderr.write("torch is not installed: _tvq_torch.so (the generation package) is not built\n")
        return
    newest = max(os.path.getmtime(TORCH_SRC), os.path.getmtime(os.path.join(INCLUDE, "tvq.h")))
    stamp, built_for = os.path.join(OBJDIR, "tvq_torch.stamp"), _torch_stamp()
    if not force and os.path.exists(TORCH_LIB) and os.path.getmtime(TORCH_LIB) >= newest and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read() == built_for:
                return
    import sysconfig

    import torch
    tmp = TORCH_LIB + ".tmp"
    torch_dir = os.path.dirname(torch.__file__)
    lib_dir = os.path.join(torch_dir, "lib")
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_tvq_torch",
           "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch._C._GLIBCXX_USE_CXX11_ABI), "-I", INCLUDE,
           "-isystem", sysconfig.get_paths()["include"], "-isystem", os.path.join(cuda, "include")]
    for d in ("include", "include/torch/csrc/api/include"):
        cmd += ["-isystem", os.path.join(torch_dir, d)]
    cmd += [TORCH_SRC, "-o", tmp, "-L", HERE, "-l:libtvq.so", "-Wl,-rpath,$ORIGIN", "-L", lib_dir, "-lc10", "-lc10_cuda",
            "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("building _tvq_torch.so failed:\n%s%s" % (r.stdout, r.stderr))
    os.replace(tmp, TORCH_LIB)
    with open(stamp, "w") as f:
        f.write(built_for)


def build(force: bool = False, verbose: bool = False) -> str:
    nvcc = _nvcc()
    os.makedirs(OBJDIR, exist_ok=True)
    newest_header = max(os.path.getmtime(h) for h in _headers())
    jobs = []
    objs = []
    for src in _sources():
        obj = os.path.join(OBJDIR, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or verbose or not os.path.exists(obj) or \
                os.path.getmtime(obj) < max(os.path.getmtime(src), newest_header):
            jobs.append((src, obj))
    if jobs:
        with cf.ThreadPoolExecutor(max_workers=min(len(jobs), os.cpu_count() or 4)) as ex:
            futs = {ex.submit(_compile, nvcc, s, o, verbose): s for s, o in jobs}
            for f in cf.as_completed(futs):
                log = f.result()
                if verbose and log:
                    sys.stderr.write("== %s\n%s" % (os.path.basename(futs[f]), log))
    if jobs or force or not os.path.exists(LIB):
        tmp = LIB + ".tmp"
        cmd = [nvcc] + ARCH + ["-shared", "-o", tmp] + objs + ["-cudart", "static"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("link failed:\n%s%s" % (r.stdout, r.stderr))
        os.replace(tmp, LIB)
    _build_torch(force)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
