"""Compiles the CUDA library in-tree: permutohedral_lattice_b200/libpl_lattice.so (sm_100a only).

    python -m permutohedral_lattice_b200.build [--force] [--verbose]

-fmad=false for pl_lattice.cu: no multiply-add contraction anywhere in the translation unit; the lattice geometry must
round every operation separately to select the same simplices as the reference CPU code.  The sources are compiled side
by side, each when it or a header is newer than its object.
"""
import os
import re
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "libpl_lattice.so")
SOURCES = [os.path.join(CSRC, "pl_lattice.cu"), os.path.join(CSRC, "channel_mix.cu")] + [
    os.path.join(CSRC, "mix_%s.cu" % part) for part in ("forward_floats", "forward_halves", "backward_floats", "backward_halves")] + [
    os.path.join(CSRC, s) for s in ("channel_norm.cu", "norm_floats.cu", "norm_halves.cu", "norm_bfloats.cu", "gated_mix.cu", "gated_floats.cu", "gated_halves.cu")]
HEADERS = [os.path.join(CSRC, h) for h in ("simplex.cuh", "common.cuh", "lattice_build.cuh", "splat.cuh",
                                             "blur_slice.cuh", "small.cuh", "export.cuh", "fp64.cuh", "direct_index.cuh", "direct_bounds.h", "crf.cuh",
                                             "smem_limit.h", "host_calls.h", "mix_common.cuh",
                                             "mix_forward.cuh", "mix_backward.cuh", "mix_tensor.cuh", "mix_tiny.cuh",
                                             "mix_host.h", "mix_launch.cuh", "mix_back_launch.cuh",
                                             "philox.cuh", "channel_norm.cuh", "norm_launch.cuh", "gated_tensor.cuh", "gated.cuh",
                                             "gated_launch.cuh", "gated_give_up.h")] + [
    os.path.join(ROOT, "include", "pl_lattice.h")]


def nvcc_path():
    for cand in (os.environ.get("CUDA_HOME"), "/usr/local/cuda"):
        if cand and os.path.exists(os.path.join(cand, "bin", "nvcc")):
            return os.path.join(cand, "bin", "nvcc")
    return "nvcc"


def _with_headers(src):
    """src and the headers that it includes, theirs included."""
    found, todo = [], [src]
    while todo:
        path = os.path.normpath(todo.pop())
        if path not in found and os.path.exists(path):
            found.append(path)
            with open(path) as f:
                todo += [os.path.join(os.path.dirname(path), name) for name in re.findall(r'^#include "([^"]+)"', f.read(), re.M)]
    return found


def build(force=False, verbose=False):
    deps = SOURCES + HEADERS
    if not force and os.path.exists(LIB) and all(os.path.getmtime(LIB) >= os.path.getmtime(d) for d in deps):
        return LIB
    flags = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC"]
    if verbose:
        flags += ["-Xptxas", "-v"]
    objects, running = [], []
    for src in SOURCES:
        obj = src[:-3] + ".o"
        objects.append(obj)
        if not force and os.path.exists(obj) and all(os.path.getmtime(obj) >= os.path.getmtime(d) for d in _with_headers(src)):
            continue
        own = ["-fmad=false"] if os.path.basename(src) == "pl_lattice.cu" else []
        running.append((obj, subprocess.Popen([nvcc_path()] + flags + own + ["-c", "-o", obj, src])))
    failed = [obj for obj, process in running if process.wait() != 0]
    for obj in failed:      # whatever is left of it is not newer than its source
        if os.path.exists(obj):
            os.remove(obj)
    if failed:
        raise RuntimeError("nvcc failed for " + ", ".join(failed))
    subprocess.check_call([nvcc_path(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", LIB] + objects)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))


HOST_TEST_SRC = os.path.join(ROOT, "tests", "helpers", "host_class_test.cpp")
HOST_TEST_BIN = os.path.join(ROOT, "tests", "helpers", "host_class_test.bin")


def build_host_class_test(force=False):
    """C++ program over include/LatticeFilterKernel.hpp used by the GPU tests (built here, runs on the
    GPU box)."""
    deps = [HOST_TEST_SRC, os.path.join(ROOT, "include", "LatticeFilterKernel.hpp"), LIB]
    if not force and os.path.exists(HOST_TEST_BIN) and all(
            os.path.getmtime(HOST_TEST_BIN) >= os.path.getmtime(d) for d in deps):
        return HOST_TEST_BIN
    cuda = os.path.dirname(os.path.dirname(nvcc_path())) if os.path.sep in nvcc_path() else "/usr/local/cuda"
    cmd = ["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(cuda, "include"),
           HOST_TEST_SRC, "-o", HOST_TEST_BIN, "-L", PKG, "-lpl_lattice", "-L", os.path.join(cuda, "lib64"),
           "-lcudart", "-Wl,-rpath,$ORIGIN/../../permutohedral_lattice_b200",
           "-Wl,-rpath," + os.path.join(cuda, "lib64")]
    subprocess.check_call(cmd)
    return HOST_TEST_BIN
