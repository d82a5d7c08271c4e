"""Builds the sm_100a shared library in-tree with nvcc.

The single library `librocm_wmma_gemm_sm100a.so` takes the place of the reference's
per-architecture `librocm_wmma_gemm_<arch>.so` objects
(rocm_wmma_gemm/CMakeLists.txt:5-93 of the reference): one target architecture, one build.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT_DIR = os.path.dirname(PKG_DIR)
LIB_NAME = "librocm_wmma_gemm_sm100a.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
# The same sources with -DB200_GEMM_TIMELINE: kernels that stamp clock values at fixed points of
# every launch (see csrc/gemm_kernels.cuh and timeline.py).  A profiling build, never loaded by
# the package itself.
TIMELINE_LIB_PATH = os.path.join(PKG_DIR, "librocm_wmma_gemm_sm100a_timeline.so")
SOURCES = [os.path.join(PKG_DIR, "csrc", "gemm_lib.cu"), os.path.join(PKG_DIR, "csrc", "epilogue_kernels.cu")]
DEPENDS = SOURCES + [
    os.path.join(PKG_DIR, "csrc", "gemm_kernels.cuh"),
    os.path.join(PKG_DIR, "csrc", "ptx_sm100.cuh"),
    os.path.join(PKG_DIR, "csrc", "config_table.inc"),
    os.path.join(PKG_DIR, "csrc", "slab_driver.inc"),
    os.path.join(PKG_DIR, "csrc", "epilogue.cuh"),
    os.path.join(PKG_DIR, "csrc", "epilogue_kernels.cuh"),
    os.path.join(PKG_DIR, "csrc", "epilogue_driver.inc"),
    os.path.join(ROOT_DIR, "include", "b200_gemm.h"),
]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-diag-suppress", "177",
]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; cannot build " + LIB_NAME)
    return exe


def is_stale(path: str = LIB_PATH) -> bool:
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    return any(os.path.getmtime(d) > t for d in DEPENDS if os.path.exists(d))


def _compile(out: str, extra: list, verbose: bool, sources: list = SOURCES) -> str:
    # one object per source, compiled side by side, then linked
    with tempfile.TemporaryDirectory() as tmp:
        objects = [os.path.join(tmp, os.path.basename(src) + ".o") for src in sources]
        cmds = [[_nvcc()] + NVCC_FLAGS + extra + (["-Xptxas", "-v"] if verbose else []) + ["-c", "-o", o, src]
                for o, src in zip(objects, sources)]
        procs = [subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for cmd in cmds]
        outputs = [p.communicate()[0] for p in procs]
        cmds.append([_nvcc()] + NVCC_FLAGS[:2] + ["-shared", "-o", out] + objects + ["-ldl"])
        if all(p.returncode == 0 for p in procs):
            link = subprocess.run(cmds[-1], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
            procs.append(link)
            outputs.append(link.stdout)
        for cmd, proc, text in zip(cmds, procs, outputs):
            if verbose:
                sys.stderr.write(text)
            if proc.returncode != 0:
                raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + text)
    return out


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the library if it is missing or older than its sources; returns its path."""
    if not force and not is_stale():
        return LIB_PATH
    return _compile(LIB_PATH, [], verbose)


def build_timeline(force: bool = False, verbose: bool = False) -> str:
    """Compile the timeline (profiling) variant of the library; returns its path."""
    if not force and not is_stale(TIMELINE_LIB_PATH):
        return TIMELINE_LIB_PATH
    # (gemm_lib.cu includes epilogue_kernels.cu in this variant: all stamps go to one set of variables)
    return _compile(TIMELINE_LIB_PATH, ["-DB200_GEMM_TIMELINE"], verbose, SOURCES[:1])


if __name__ == "__main__":
    if "--timeline" in sys.argv:
        print(build_timeline(force="--force" in sys.argv, verbose="-v" in sys.argv))
    else:
        print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
