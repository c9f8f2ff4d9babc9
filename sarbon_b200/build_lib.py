"""Build ``libsarbon_sparse.so`` (the C ABI in ``include/sarbon_sparse.h``) for sm_100a, and ``_paged_calls``, the
Python module through which the paged memory's calls reach it with little host time.  The library needs neither Python nor
torch; where the module cannot be built, the Python side makes its calls.

The library is built in-tree next to this file so that it travels with the source
tree; object files go to ``sarbon_b200/_build``.  Usage::

    python -m sarbon_b200.build_lib          # or: from sarbon_b200.build_lib import build
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OBJ = PKG / "_build"
LIB = PKG / "libsarbon_sparse.so"
# (named for its interpreter: no other one looks at it)
CALLS_SOURCE, CALLS_LIB = CSRC / "sb_paged_calls.cpp", PKG / f"_paged_calls{sysconfig.get_config_var('EXT_SUFFIX')}"
CALLS_FOR = OBJ / "paged_calls_built_for.txt"  # the torch that it was built against
SOURCES = ["sb_engine.cu", "sb_gate.cu", "sb_conv_tc.cu", "sb_conv_simt.cu", "sb_noalloc.cu", "sb_cells.cu", "sb_boxes.cu",
           "sb_prep.cu", "sb_deform.cu", "sb_gemm.cu", "sb_detops.cu", "sb_attn.cu", "sb_xattn.cu", "sb_xattn_few.cu", "sb_xattn_bwd.cu",
           "sb_rope.cu", "sb_gnorm.cu", "sb_paged_attn.cu", "sb_paged_cache.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
         "--expt-relaxed-constexpr", f"-I{PKG.parent / 'include'}"]


def nvcc() -> str:
    for c in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if c and Path(c).exists():
            return c
    raise RuntimeError("nvcc not found")


def _compile(src: str, extra) -> Path:
    out = OBJ / (Path(src).stem + ".o")
    cmd = [nvcc(), *ARCH, *FLAGS, *extra, "-c", str(CSRC / src), "-o", str(out)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    if r.stderr.strip():
        sys.stderr.write(r.stderr)
    return out


def _run(what, cmd):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")


def build_calls(force: bool = False, verbose: bool = False) -> Path:
    """Compile the Python module against the installed torch."""
    import torch
    header = PKG.parent / "include" / "sarbon_sparse.h"
    root = Path(torch.__file__).resolve().parent
    newest = max(p.stat().st_mtime for p in (CALLS_SOURCE, header))
    if not force and CALLS_LIB.exists() and CALLS_LIB.stat().st_mtime > newest and CALLS_FOR.exists() and \
            CALLS_FOR.read_text() == torch.__version__:
        return CALLS_LIB
    cuda = Path(nvcc()).resolve().parents[1]
    found = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", sysconfig.get_paths()["include"],
             cuda / "include"]
    tmp = CALLS_LIB.with_suffix(".so.tmp")
    _run("g++", ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-I{header.parent}",
                 f'-DSB_BUILT_FOR="{torch.__version__}"', *(x for p in found for x in ("-isystem", str(p))), str(CALLS_SOURCE),
                 "-o", str(tmp), f"-L{root / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"])
    os.replace(tmp, CALLS_LIB)
    OBJ.mkdir(exist_ok=True)
    CALLS_FOR.write_text(torch.__version__)
    if verbose:
        print(f"built {CALLS_LIB}")
    return CALLS_LIB


def build(force: bool = False, extra=(), verbose: bool = False) -> Path:
    """Build the shared library, then the Python module, without which all goes on."""
    lib = build_library(force, extra, verbose)
    for old in PKG.glob("_paged_calls*.so"):
        if old != CALLS_LIB:  # another interpreter's, or of no interpreter's name, against other declarations
            old.unlink()
    try:
        build_calls(force, verbose)
    except (RuntimeError, OSError, ImportError) as e:
        CALLS_LIB.unlink(missing_ok=True)  # what is there was built for something else
        warnings.warn(f"_paged_calls was not built, small calls of the paged memory take longer on the host: {e}", RuntimeWarning)
    return lib


def build_library(force: bool = False, extra=(), verbose: bool = False) -> Path:
    """Compile every CUDA source for sm_100a and link the shared library."""
    srcs = [CSRC / s for s in SOURCES] + list(CSRC.glob("*.cuh")) + [PKG.parent / "include" / "sarbon_sparse.h"]
    if LIB.exists() and not force:
        newest = max(p.stat().st_mtime for p in srcs)
        if LIB.stat().st_mtime > newest:
            return LIB
    OBJ.mkdir(exist_ok=True)
    with ThreadPoolExecutor(len(SOURCES)) as ex:
        objs = list(ex.map(lambda s: _compile(s, list(extra)), SOURCES))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH, "-shared", "--cudart", "static", "-o", str(tmp), *map(str, objs)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
