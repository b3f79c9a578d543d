"""Builds ``libaarambh_b200.so`` in-tree with nvcc for sm_100a.

Usage: ``python aarambh-ai_b200/build.py [--force] [--verbose]``.  One object per
``csrc/*.cu`` (compiled in parallel, skipped when newer than its sources), then
one shared library next to this file.  nvcc cross-compiles without a GPU.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libaarambh_b200.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC,-fvisibility=hidden", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC,
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def _newest(paths) -> float:
    return max(os.path.getmtime(p) for p in paths)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    headers = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(ROOT, "include", "*.h"))
    hdr_time = _newest(headers) if headers else 0.0
    jobs = []
    objects = []
    for src in sources:
        obj = os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")
        objects.append(obj)
        if force or not os.path.exists(obj) or os.path.getmtime(obj) < max(os.path.getmtime(src), hdr_time):
            cmd = [_nvcc()] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", src, "-o", obj]
            jobs.append(cmd)

    def run(cmd):
        res = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, res

    with cf.ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as pool:
        for cmd, res in pool.map(run, jobs):
            if verbose or res.returncode != 0:
                sys.stderr.write(" ".join(cmd) + "\n" + res.stdout + res.stderr)
            if res.returncode != 0:
                raise RuntimeError("nvcc failed for " + cmd[-3])
    if jobs or not os.path.exists(LIB):
        link = [_nvcc(), "-shared", "-o", LIB] + objects + ["-lcudart", "-ldl"]
        res = subprocess.run(link, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("link of libaarambh_b200.so failed")
    try:
        build_fast(force, verbose)
    except (RuntimeError, OSError) as e:   # no torch, no headers of it or of Python, no compiler: the library is whole without it
        if os.path.exists(FAST):   # made for another torch, Python or header
            os.remove(FAST)
        sys.stderr.write(f"_fast.so is not built, calls of a serving step take some 8 us more on the host: {e}\n")
    return LIB


FAST = os.path.join(HERE, "_fast.so")


def build_fast(force: bool = False, verbose: bool = False) -> str:
    """csrc/fast.cpp, the Python module of the serving step's plain calls, against the torch and the Python that run this.  dispatch.py does without it."""
    import importlib.util
    import sysconfig
    spec = importlib.util.find_spec("torch")
    if spec is None:
        raise RuntimeError("torch is needed to build _fast.so")
    torch_dir, source, header = os.path.dirname(spec.origin), os.path.join(CSRC, "fast.cpp"), os.path.join(ROOT, "include", "aarambh_b200.h")
    if not force and os.path.exists(FAST) and os.path.getmtime(FAST) >= _newest([source, header, os.path.join(torch_dir, "version.py")]):
        return FAST
    cuda = os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-shared", source, "-o", FAST + ".new", "-I" + os.path.join(ROOT, "include"),
           "-I" + os.path.join(torch_dir, "include"), "-I" + os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"), "-I" + cuda,
           "-I" + sysconfig.get_path("include"), "-L" + os.path.join(torch_dir, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda",
           "-L" + HERE, "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(" ".join(cmd) + "\n" + res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError("g++ failed for fast.cpp")
    os.replace(FAST + ".new", FAST)
    return FAST


def build_locked() -> str:
    """``build`` under a file lock, for programs that may start together in a fresh checkout."""
    import fcntl
    os.makedirs(OBJ, exist_ok=True)
    with open(os.path.join(OBJ, ".lock"), "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        return build()


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
