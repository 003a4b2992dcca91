"""Build the detkernels_b200 shared library (sm_100a) in-tree.

    python -m detkernels_b200.build          # -> detkernels_b200/libdetkernels_b200.so

The library is four CUDA translation units (csrc/*.cu), compiled side by side
with nvcc for `sm_100a` only.  It links the CUDA runtime statically and reaches the
driver API (tensor-map encoding) through cudaGetDriverEntryPointByVersion, so
the .so loads on a machine without a GPU driver (symbol checks, CPU tests).
"""
from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sys
import tempfile

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(os.path.dirname(PKG_DIR), "include")
LIB_NAME = "libdetkernels_b200.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
STAMP_PATH = LIB_PATH + ".srchash"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _sources():
    files = []
    for d in (CSRC, INCLUDE):
        for name in sorted(os.listdir(d)):
            if name.endswith((".cu", ".cuh", ".h")):
                files.append(os.path.join(d, name))
    return files


def source_hash() -> str:
    h = hashlib.sha256()
    for path in _sources():
        h.update(os.path.basename(path).encode())
        with open(path, "rb") as f:
            h.update(f.read())
    h.update(" ".join(NVCC_FLAGS).encode())
    return h.hexdigest()


def nvcc_path() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the detkernels_b200 library needs the CUDA toolkit to build")


def is_up_to_date() -> bool:
    if not os.path.exists(LIB_PATH) or not os.path.exists(STAMP_PATH):
        return False
    with open(STAMP_PATH) as f:
        return f.read().strip() == source_hash()


def _run(cmds, verbose):
    """Run commands side by side; raises with their output if one fails."""
    procs = []
    for cmd in cmds:
        if verbose:
            print("[detkernels_b200] " + " ".join(cmd), flush=True)
        procs.append(subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True))
    outs = [p.communicate()[0] for p in procs]
    if any(p.returncode for p in procs):
        sys.stderr.write("".join(o for p, o in zip(procs, outs) if p.returncode))
        raise RuntimeError("nvcc failed building %s" % LIB_NAME)


def build(force: bool = False, verbose: bool = True) -> str:
    """Compile csrc/*.cu into LIB_PATH unless it is already current."""
    if not force and is_up_to_date():
        return LIB_PATH
    tmp = LIB_PATH + ".tmp"
    units = [os.path.join(CSRC, name) for name in sorted(os.listdir(CSRC)) if name.endswith(".cu")]
    with tempfile.TemporaryDirectory() as obj_dir:
        objs = [os.path.join(obj_dir, os.path.basename(u) + ".o") for u in units]
        _run([[nvcc_path(), *NVCC_FLAGS, "-I", INCLUDE, "-c", "-o", o, u] for u, o in zip(units, objs)], verbose)
        _run([[nvcc_path(), *NVCC_FLAGS, "-shared", "-o", tmp, *objs]], verbose)
    os.replace(tmp, LIB_PATH)
    with open(STAMP_PATH, "w") as f:
        f.write(source_hash())
    return LIB_PATH


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB_PATH)
