"""Builds libbtp_sm100.so (the C-ABI library with the sm_100a kernels) in-tree with nvcc.

    python -m spear_b200.build [--force] [--verbose]

The result lands next to this file as spear_b200/lib/libbtp_sm100.so.  nvcc cross-compiles, so no
GPU is needed to build.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libbtp_sm100.so")
SOURCES = [os.path.join(CSRC, "btp_sm100.cu"), os.path.join(CSRC, "norm_sm100.cu"),
           os.path.join(CSRC, "conv_sm100.cu"), os.path.join(CSRC, "scan_sm100.cu")]
HEADERS = [
    os.path.join(CSRC, "btp_kernels.cuh"),
    os.path.join(CSRC, "btp_decode.cuh"),
    os.path.join(CSRC, "btp_gated.cuh"),
    os.path.join(CSRC, "btp_gated_bwd.cuh"),
    os.path.join(CSRC, "btp_ptx.cuh"),
    os.path.join(CSRC, "btp_host.cuh"),
    os.path.join(CSRC, "btp_elem.cuh"),
    os.path.join(CSRC, "elem_host.cuh"),
    os.path.join(CSRC, "norm_kernels.cuh"),
    os.path.join(CSRC, "conv_kernels.cuh"),
    os.path.join(CSRC, "scan_kernels.cuh"),
    os.path.join(CSRC, "scan_bwd_kernels.cuh"),
    os.path.join(CSRC, "sum_kernels.cuh"),
    os.path.join(os.path.dirname(HERE), "include", "btp_sm100.h"),
]


def nvcc_path() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found; set NVCC or put it on PATH")
    return cand


def is_stale() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    built = os.path.getmtime(LIB_PATH)
    return any(os.path.getmtime(p) > built for p in SOURCES + HEADERS)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile for sm_100a only.  Returns the path of the shared library."""
    if not force and not is_stale():
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    flags = [
        "-gencode", "arch=compute_100a,code=sm_100a",
        "-O3", "-std=c++17", "-lineinfo",
        "-Xcompiler", "-fPIC",
        "-Xptxas", "-v" if verbose else "-O3",
    ]
    objects = [os.path.join(LIB_DIR, os.path.splitext(os.path.basename(p))[0] + ".o") for p in SOURCES]
    newest_header = max(os.path.getmtime(p) for p in HEADERS)
    running = []
    for src, obj in zip(SOURCES, objects):  # the translation units compile side by side
        if not force and os.path.exists(obj) and os.path.getmtime(obj) > max(newest_header, os.path.getmtime(src)):
            continue
        cmd = [nvcc_path(), *flags, "-c", "-o", obj, src]
        running.append((cmd, obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)))
    failed = []
    for cmd, obj, proc in running:
        out, err = proc.communicate()
        if verbose:
            sys.stderr.write(err)
        if proc.returncode != 0:
            if os.path.exists(obj):
                os.remove(obj)
            failed.append("nvcc failed:\n" + " ".join(cmd) + "\n" + out + err)
    if failed:
        raise RuntimeError("\n".join(failed))
    cmd = [nvcc_path(), *flags[:2], "-shared", "-Xcompiler", "-fPIC", "-o", LIB_PATH, *objects]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + proc.stdout + proc.stderr)
    return LIB_PATH


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(path)
