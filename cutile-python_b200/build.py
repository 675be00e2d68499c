"""Builds libb200k.so (sm_100a only) from csrc/*.cu with nvcc, and the host module _plans.so from
csrc/launch_plans.cpp, in-tree.

Usage:  python cutile-python_b200/build.py [--force] [--verbose]

Each translation unit is compiled to an object file in parallel and the objects are
linked into ``b200k/libb200k.so`` next to the Python package, so the shared library
travels with the source tree.  Only ``-gencode arch=compute_100a,code=sm_100a`` is
used: the tcgen05 instructions do not exist on any other target.
"""
from __future__ import annotations

import argparse
import concurrent.futures
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ_DIR = os.path.join(HERE, "build")
LIB_PATH = os.path.join(HERE, "b200k", "libb200k.so")
PLANS_SRC = os.path.join(CSRC, "launch_plans.cpp")
PLANS_PATH = os.path.join(HERE, "b200k", "_plans.so")
PLANS_STAMP = os.path.join(OBJ_DIR, "_plans.stamp")      # what _plans.so was built with

NVCC_FLAGS = [
    "-std=c++17", "-O3", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; the library cannot be built")
    return exe


def _sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers() -> list[str]:
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hdrs.append(os.path.join(HERE, "..", "include", "b200k.h"))
    return hdrs


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _plans_command(nvcc: str) -> list[str]:
    """The host module: CPython and torch headers, against the libraries `import torch` loads."""
    torch = importlib.util.find_spec("torch").submodule_search_locations[0]
    include = os.path.join(torch, "include")
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc)))
    return [shutil.which("g++") or "g++", "-std=c++17", "-O2", "-fPIC", "-shared", PLANS_SRC, "-o", PLANS_PATH,
            "-I", include, "-I", os.path.join(include, "torch", "csrc", "api", "include"),
            "-I", os.path.join(cuda, "include"), "-I", sysconfig.get_paths()["include"],
            "-L", os.path.join(torch, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]


def _plans_stamp(nvcc: str) -> str:
    """What the host module depends on besides its source: the command, this interpreter and the
    torch whose classes it uses (they change their layout without changing their path)."""
    return "\n".join([*_plans_command(nvcc), sys.version, importlib.metadata.version("torch")])


def _plans_stale(nvcc: str) -> bool:
    if _stale(PLANS_PATH, [PLANS_SRC]) or not os.path.exists(PLANS_STAMP):
        return True
    with open(PLANS_STAMP) as f:
        return f.read() != _plans_stamp(nvcc)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ_DIR, exist_ok=True)
    nvcc = _nvcc()
    hdrs = _headers()
    jobs = []
    objs = []
    plans = force or _plans_stale(nvcc)
    if plans:
        jobs.append(_plans_command(nvcc))
    for src in _sources():
        obj = os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or _stale(obj, [src] + hdrs):
            cmd = [nvcc, *NVCC_FLAGS, "-c", src, "-o", obj]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, r

    if jobs:
        with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(jobs))) as pool:
            for cmd, r in pool.map(run, jobs):
                if verbose or r.returncode != 0:
                    sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
                if r.returncode != 0:
                    raise RuntimeError(f"compiling failed: {' '.join(cmd)}")
    if plans:
        with open(PLANS_STAMP, "w") as f:
            f.write(_plans_stamp(nvcc))
    if jobs or force or _stale(LIB_PATH, objs):
        cmd = [nvcc, "-shared", "-o", LIB_PATH, *objs, "-cudart", "static"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    return LIB_PATH


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
