"""Builds libfast_moss_b200.so (sm_100a) in-tree with nvcc, and the package's
native calls (_binding-<torch>-<python>.so) with the host compiler.

Usage: python build.py [--force]

Both are written next to the Python package (fast_moss_b200/) so that they
are found without any installation step and travel with the source tree.  The
library comes first and needs only the CUDA toolkit; the binding needs torch's
and Python's headers, and is left out where torch is not installed.
"""

import argparse
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
PACKAGE = os.path.join(HERE, "fast_moss_b200")
LIB = os.path.join(PACKAGE, "libfast_moss_b200.so")
BINDING_SOURCE = os.path.join(CSRC, "binding.cpp")
SOURCES = ["capi.cu", "layer_norm.cu", "rope.cu", "gated_act.cu", "lfq.cu", "rvq.cu",
           "rvq_tc.cu", "rvq_pair.cu", "rvq_noalloc.cu", "qkv_rope.cu", "history_attn.cu", "linear.cu",
           "lfq_rvq.cu", "qk_norm_rope.cu", "paged_attn.cu", "paged_attn_tc.cu"]

# Compiled as a whole program each (no device symbols shared with the others):
# setmaxnreg is ignored in relocatable device code.
STANDALONE = ["paged_attn_tc.cu"]

NVCC_FLAGS = [
    "-O3",
    "-std=c++17",
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-Xcompiler",
    "-fPIC",
    "-Xcompiler",
    "-fvisibility=hidden",
]


def nvcc_path():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; the CUDA toolkit is required to build fast_moss_b200")


def inputs():
    files = [os.path.join(CSRC, s) for s in SOURCES]
    files += [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cuh")]
    files += [os.path.join(INCLUDE, "fast_moss_b200.h"), os.path.abspath(__file__)]
    return files


def up_to_date(target, files=None):
    if not os.path.exists(target):
        return False
    built = os.path.getmtime(target)
    return all(os.path.getmtime(f) <= built for f in files or inputs())


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed to build fast_moss_b200")


def torch_directory():
    """Where torch is installed, None where it is not (it is not imported)."""
    spec = importlib.util.find_spec("torch")
    return os.path.dirname(spec.origin) if spec and spec.origin else None


def torch_version():
    """torch.__version__ of the installed torch, which is not imported."""
    with open(os.path.join(torch_directory(), "version.py")) as f:
        return re.search(r"^__version__ *= *['\"]([^'\"]+)", f.read(), flags=re.M).group(1)


def binding_path():
    """The binding's file.  It is built against one torch and one Python and
    fits no other, so it is named for both (fast_moss_b200._lib.binding_path)."""
    return os.path.join(PACKAGE, f"_binding-{torch_version()}-{sys.implementation.cache_tag}.so")


def binding_command(out):
    torch = torch_directory()
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc_path())))
    headers = [os.path.join(torch, "include"), os.path.join(cuda, "include"), INCLUDE,
               sysconfig.get_paths()["include"]]
    libs = ["torch_python", "torch", "torch_cpu", "torch_cuda", "c10", "c10_cuda"]
    return [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-Wall", "-fPIC", "-shared",
            "-fvisibility=hidden", *(f"-I{h}" for h in headers), BINDING_SOURCE, "-o", out,
            "-L" + os.path.join(torch, "lib"), *(f"-l{name}" for name in libs)]


def build_binding(force=False, verbose=False):
    files = [BINDING_SOURCE, os.path.join(INCLUDE, "fast_moss_b200.h"), os.path.abspath(__file__)]
    target = binding_path()
    if force or not up_to_date(target, files):
        _run(binding_command(target + ".tmp"), verbose)
        os.replace(target + ".tmp", target)


def build(force=False, verbose=False):
    """Compiles the CUDA sources into the shared library, and the binding where
    torch is installed; returns the library's path."""
    if force or not up_to_date(LIB):
        build_library(verbose)
    if torch_directory():
        build_binding(force, verbose)
    else:
        sys.stderr.write("torch not found: the library is built, the Python package's native "
                         "calls are not\n")
    return LIB


def build_library(verbose=False):
    tmp = LIB + ".tmp"
    with tempfile.TemporaryDirectory() as work:
        objects = [os.path.join(work, s[:-3] + ".o") for s in SOURCES]
        compiles = []
        for source, obj in zip(SOURCES, objects):
            kind = ["-DMOSS_STANDALONE"] if source in STANDALONE else ["-rdc=true"]
            compiles.append([nvcc_path(), *NVCC_FLAGS, *kind, "-I", INCLUDE, "-c",
                             os.path.join(CSRC, source), "-o", obj])
        with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
            list(pool.map(lambda cmd: _run(cmd, verbose), compiles))
        _run([nvcc_path(), *NVCC_FLAGS, "-shared", *objects, "-o", tmp], verbose)
    os.replace(tmp, LIB)


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--force", action="store_true")
    args = parser.parse_args()
    print(build(force=args.force, verbose=True))
