"""Build libturboadam_b200.so (sm_100a) in-tree.

    python -m turboadam_b200.csrc.build [--verbose-ptxas]

Each source is compiled to an object of its own (csrc/_build/, rebuilt when
the source or a header it includes is newer) and the objects are linked.

Flags that make the packed step's device arithmetic bit-identical to the host
checker: --fmad=false (no a*b+c contraction; the sources call __fmaf_rn
explicitly where torch fuses), IEEE division and square root, no flush-to-zero.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
OUT = os.path.join(PKG, "libturboadam_b200.so")
OBJ_DIR = os.path.join(HERE, "_build")
INCLUDE = os.path.join(os.path.dirname(PKG), "include")


def _paths(*names):
    return [os.path.join(HERE, f) for f in names]


# source -> the headers it includes
UNITS = {
    os.path.join(HERE, "ta_api.cu"):
        _paths("ta_kernels.cuh", "ta_codec.cuh", "ta_device.cuh", "ta_math.h", "ta_host.h")
        + [os.path.join(INCLUDE, "turboadam_b200.h")],
    os.path.join(HERE, "ta_mx_api.cu"):
        _paths("ta_mx_device.cuh", "ta_mx_product.cuh", "ta_mx_chain.cuh", "ta_mx_elementwise.cuh", "ta_mx_few.cuh",
                  "ta_host.h")
        + [os.path.join(INCLUDE, "turboadam_b200.h"),
           os.path.join(INCLUDE, "turboadam_b200_matrix.h")],
}
SOURCES = list(UNITS)
DEPS = sorted({f for src, heads in UNITS.items() for f in [src, *heads]})


def nvcc() -> str:
    for c in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def flags(ptxas_verbose: bool = False) -> list[str]:
    f = [
        "-gencode", "arch=compute_100a,code=sm_100a",
        "-O3", "-lineinfo", "-std=c++17",
        "--fmad=false", "-prec-div=true", "-prec-sqrt=true", "-ftz=false",
        "-Xcompiler", "-fPIC,-ffp-contract=off,-fvisibility=hidden",
        "-shared", "-cudart", "static",
    ]
    if ptxas_verbose:
        f += ["-Xptxas", "-v"]
    return f


def up_to_date() -> bool:
    if not os.path.exists(OUT):
        return False
    t = os.path.getmtime(OUT)
    return all(os.path.getmtime(d) <= t for d in DEPS)


def _object(src: str) -> str:
    return os.path.join(OBJ_DIR, os.path.splitext(os.path.basename(src))[0] + ".o")


def _stale(src: str) -> bool:
    obj = _object(src)
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    return any(os.path.getmtime(d) > t for d in [src, *UNITS[src]])


def build(force: bool = False, ptxas_verbose: bool = False, quiet: bool = False) -> str:
    if not force and up_to_date():
        return OUT
    os.makedirs(OBJ_DIR, exist_ok=True)
    base = [f for f in flags(ptxas_verbose) if f != "-shared"]
    jobs = []
    for src in SOURCES:
        if force or _stale(src):
            tmp = _object(src) + ".tmp.o"
            cmd = [nvcc()] + base + ["-c", "-o", tmp, src]
            if not quiet:
                print(" ".join(cmd), flush=True)
            jobs.append((src, tmp, cmd, subprocess.Popen(cmd)))
    for src, tmp, cmd, job in jobs:
        if job.wait() != 0:
            raise subprocess.CalledProcessError(job.returncode, cmd)
        os.replace(tmp, _object(src))
    tmp = OUT + ".tmp"
    cmd = [nvcc()] + flags() + ["-o", tmp] + [_object(src) for src in SOURCES]
    if not quiet:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose-ptxas", action="store_true")
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    build(force=a.force or a.verbose_ptxas, ptxas_verbose=a.verbose_ptxas)
    sys.exit(0)
