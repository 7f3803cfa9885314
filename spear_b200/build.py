"""Builds libbtp_sm100.so (the C-ABI library with the sm_100a kernels) in-tree with nvcc, and beside it btp_torch.so, the
Python module of the token-major operators on torch tensors (host C++ against torch's headers, on top of the C ABI).

    python -m spear_b200.build [--force] [--verbose]

The results land next to this file in spear_b200/lib.  nvcc cross-compiles, so no
GPU is needed to build.
"""

from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libbtp_sm100.so")
MODULE_PATH = os.path.join(LIB_DIR, "btp_torch.so")
MODULE_SOURCE = os.path.join(CSRC, "btp_torch.cpp")
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
    if not os.path.exists(LIB_PATH) or not os.path.exists(MODULE_PATH):
        return True
    built, made = os.path.getmtime(LIB_PATH), os.path.getmtime(MODULE_PATH)
    return any(os.path.getmtime(p) > built for p in SOURCES + HEADERS) or os.path.getmtime(MODULE_SOURCE) > made


def module_commands(obj: str) -> tuple[list[str], list[str]]:
    """The compile and the link command of btp_torch.so."""
    torch = os.path.join(importlib.util.find_spec("torch").submodule_search_locations[0])
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc_path())))
    includes = [os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"),
                os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    compiler = os.environ.get("CXX") or "g++"
    compile_it = [compiler, "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=btp_torch",
                  *(f for i in includes for f in ("-isystem", i)), "-c", "-o", obj, MODULE_SOURCE]
    link_it = [compiler, "-shared", "-o", MODULE_PATH, obj, "-L" + os.path.join(torch, "lib"), "-ltorch", "-ltorch_cpu", "-ltorch_cuda",
               "-lc10", "-lc10_cuda", "-ltorch_python", "-L" + LIB_DIR, "-l:libbtp_sm100.so", "-Wl,-rpath,$ORIGIN"]
    return compile_it, link_it


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
    host_obj = os.path.join(LIB_DIR, "btp_torch.o")
    compile_it, link_it = module_commands(host_obj)
    if force or not os.path.exists(host_obj) or os.path.getmtime(host_obj) < max(os.path.getmtime(MODULE_SOURCE), os.path.getmtime(HEADERS[-1])):
        running.append((compile_it, host_obj, subprocess.Popen(compile_it, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)))
    failed = []
    for cmd, obj, proc in running:
        out, err = proc.communicate()
        if verbose:
            sys.stderr.write(err)
        if proc.returncode != 0:
            if os.path.exists(obj):
                os.remove(obj)
            failed.append("the compiler failed:\n" + " ".join(cmd) + "\n" + out + err)
    if failed:
        raise RuntimeError("\n".join(failed))
    for cmd in ([nvcc_path(), *flags[:2], "-shared", "-Xcompiler", "-fPIC", "-o", LIB_PATH, *objects], link_it):
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError("linking failed:\n" + " ".join(cmd) + "\n" + proc.stdout + proc.stderr)
    return LIB_PATH


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(path)
