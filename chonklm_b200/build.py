"""Build the CUDA engine library `libchonk_b200.so` in-tree for sm_100a.

Plain nvcc, no torch extension: the library exports only the C ABI declared
in include/chonk_b200.h and links the CUDA runtime statically.
"""
from __future__ import annotations

import glob
import os
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
LIB = os.path.join(PKG, "libchonk_b200.so")
OBJ = os.path.join(PKG, "_build")
ABI = os.path.join(ROOT, "include", "chonk_b200.h")
KV = sorted(glob.glob(os.path.join(PKG, "csrc", "ck_kv*"))) + [os.path.join(PKG, "csrc", "ck_ptx.cuh"), ABI]
DEPS = sorted(glob.glob(os.path.join(PKG, "csrc", "*.cu*"))) + [os.path.join(PKG, "csrc", "ck_kv.h"), ABI]
# translation units and what each is rebuilt for
SOURCES = {os.path.join(PKG, "csrc", "ck_engine.cu"): [p for p in DEPS if not os.path.basename(p).startswith("ck_kv") or
                                                       p.endswith(".h")],
           os.path.join(PKG, "csrc", "ck_kv.cu"): KV}
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
         "-cudart", "static"]


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(p) > t for p in DEPS)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    tmp = LIB + f".tmp{os.getpid()}"
    running, objects = [], []
    for src, deps in SOURCES.items():   # one nvcc per stale unit, side by side
        obj = os.path.join(OBJ, os.path.basename(src) + ".o")
        objects.append(obj)
        if not force and os.path.exists(obj) and all(os.path.getmtime(p) <= os.path.getmtime(obj) for p in deps):
            continue
        part = obj + f".tmp{os.getpid()}"
        cmd = [NVCC, *FLAGS, "-c", "-o", part, src]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd), file=sys.stderr)
        running.append((subprocess.Popen(cmd), cmd, part, obj))
    for p, cmd, part, obj in running:
        if p.wait():
            raise subprocess.CalledProcessError(p.returncode, cmd)
        os.replace(part, obj)
    subprocess.check_call([NVCC, *FLAGS, "-shared", "-o", tmp, *objects])
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
