"""Build recipe of the CUDA library: nvcc, sm_100a only, output in-tree next to this file."""
from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "liblinmt_decoder.so")
TORCH_LIB = os.path.join(HERE, "_device_ops.so")     # the operators' front for torch tensors (device_ops)
SOURCES = ["engine.cu", "engine_tc.cu", "frontend.cu", "kernel_entry.cu", "noalloc_entry.cu", "beam_ops.cu", "pages4_ops.cu",
           "pages4_attend.cu", "pages8_ops.cu", "pages8_attend.cu", "page_ops.cu", "token_ops.cu", "unk_post.cpp"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC,-fopenmp,-O3", "--use_fast_math=false"]


def _newest_source() -> float:
    t = 0.0
    for root in (CSRC, os.path.join(HERE, "..", "include")):
        for fn in os.listdir(root):
            if fn == "device_ops_torch.cpp":      # not part of the library
                continue
            t = max(t, os.path.getmtime(os.path.join(root, fn)))
    return t


def torch_front_is_built() -> bool:
    return os.path.exists(TORCH_LIB)


def _build_torch_front(force: bool, verbose: bool):
    """Starts the compiler on the front for torch tensors; (command, process) or None where it is up to date or torch is not installed.  It calls the library's
    C ABI and is found beside it."""
    src = os.path.join(CSRC, "device_ops_torch.cpp")
    newest = max(os.path.getmtime(src), os.path.getmtime(os.path.join(HERE, "..", "include", "linmt_decoder.h")))
    if not force and os.path.exists(TORCH_LIB) and os.path.getmtime(TORCH_LIB) >= newest:
        return None
    spec = importlib.util.find_spec("torch")
    if spec is None:
        return None
    torch_dir = spec.submodule_search_locations[0]
    cuda = os.path.dirname(os.path.dirname(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"))
    lib = os.path.join(torch_dir, "lib")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-I" + os.path.join(torch_dir, "include"), "-I" + os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
           "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(cuda, "include"), src, "-o", TORCH_LIB, "-L" + HERE, "-llinmt_decoder", "-L" + lib, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda",
           "-ltorch_python", "-Wl,-rpath,$ORIGIN", "-Wl,-rpath," + lib] + (["-v"] if verbose else [])
    return cmd, subprocess.Popen(cmd)


def build(force: bool = False, verbose: bool = False) -> str:
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < _newest_source():
        _build_library(verbose)
    front = _build_torch_front(force, verbose)
    if front and front[1].wait() != 0:
        raise RuntimeError("g++ failed: " + " ".join(front[0]))
    return LIB


def _build_library(verbose: bool) -> None:
    objs = []
    procs = []
    os.makedirs(os.path.join(HERE, "build"), exist_ok=True)
    for src in SOURCES:
        obj = os.path.join(HERE, "build", os.path.splitext(src)[0] + ".o")
        cmd = ["nvcc"] + [f for f in NVCC_FLAGS if not f.startswith("--use_fast_math")] + \
              (["-Xptxas", "-v"] if verbose else []) + ["-c", os.path.join(CSRC, src), "-o", obj]
        procs.append((cmd, subprocess.Popen(cmd)))
        objs.append(obj)
    for cmd, p in procs:
        if p.wait() != 0:
            raise RuntimeError("nvcc failed: " + " ".join(cmd))
    link = ["nvcc", "-shared", "-o", LIB] + objs + ["-Xcompiler", "-fopenmp", "-lcudart", "-lcuda"]
    subprocess.run(link, check=True)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
