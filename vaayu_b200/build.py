"""Build libvaayu_b200.so from vaayu_b200/csrc/*.cu with nvcc for sm_100a, in-tree, and the dense
layers' host extension (_dense_host.so, csrc/dense_host.cpp) with g++ against torch.

    python -m vaayu_b200.build [--force] [--verbose]

Objects go to vaayu_b200/_build/, the library to vaayu_b200/libvaayu_b200.so (both git-ignored;
the built library is what the Python package loads, so it travels with the source tree).
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
SRC = PKG / "csrc"
OBJ = PKG / "_build"
LIB = PKG / "libvaayu_b200.so"
INCLUDE = PKG.parent / "include"
HOST_SRC = SRC / "dense_host.cpp"
HOST_LIB = PKG / "_dense_host.so"
HOST_MADE = OBJ / "_dense_host.txt"      # what it was built with

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-O3",
         "--expt-relaxed-constexpr", f"-I{INCLUDE}"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is needed to build libvaayu_b200")


def _headers_mtime() -> float:
    hs = list(SRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    return max((h.stat().st_mtime for h in hs), default=0.0)


def _compile(src: Path, verbose: bool, ptxas_v: bool) -> Path:
    obj = OBJ / (src.stem + ".o")
    cmd = [nvcc(), *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
    if ptxas_v:
        cmd += ["-Xptxas", "-v"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stderr}")
    if verbose and res.stderr.strip():
        print(res.stderr)
    return obj


def build_host(force: bool = False) -> Path:
    """The extension module that makes the dense layers' ordinary calls without Python in between."""
    import platform
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    flags = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{root / 'include'}",
             f"-I{root / 'include/torch/csrc/api/include'}", f"-I{cuda / 'include'}",
             f"-I{sysconfig.get_paths()['include']}", f"-L{root / 'lib'}",
             # the C++ library of the process, by its file: a toolchain that has only the archive would put a
             # second one into the extension, whose streams crash on the first error message with a number
             "-l:libstdc++.so.6", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python"]
    # it links against one torch and one Python: another of either, or other flags, makes it stale
    made_with = "\n".join([f"torch {torch.__version__}", f"python {platform.python_version()}", *flags])
    newest = max(HOST_SRC.stat().st_mtime, *(h.stat().st_mtime for h in INCLUDE.glob("*.h")))
    if (not force and HOST_LIB.exists() and HOST_LIB.stat().st_mtime >= newest and HOST_MADE.exists()
            and HOST_MADE.read_text() == made_with):
        return HOST_LIB
    tmp = HOST_LIB.with_suffix(".so.tmp%d" % os.getpid())
    libs = [f for f in flags if f.startswith("-l")]      # behind the source, which needs them
    cmd = [*(f for f in flags if f not in libs), str(HOST_SRC), "-o", str(tmp), *libs]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{HOST_SRC.name} failed to build:\n{res.stderr}")
    os.replace(tmp, HOST_LIB)
    OBJ.mkdir(exist_ok=True)
    HOST_MADE.write_text(made_with)
    return HOST_LIB


def build(force: bool = False, verbose: bool = False, ptxas_v: bool = False) -> Path:
    """Compile every stale .cu (in parallel) and link the shared library; returns its path."""
    OBJ.mkdir(exist_ok=True)
    sources = sorted(SRC.glob("*.cu"))
    hdr = _headers_mtime()
    stale = [s for s in sources
             if force or ptxas_v or not (OBJ / (s.stem + ".o")).exists()
             or (OBJ / (s.stem + ".o")).stat().st_mtime < max(s.stat().st_mtime, hdr)]
    if stale:
        with ThreadPoolExecutor(max_workers=min(8, len(stale))) as ex:
            list(ex.map(lambda s: _compile(s, verbose, ptxas_v), stale))
    objs = [OBJ / (s.stem + ".o") for s in sources]
    if stale or not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        tmp = LIB.with_suffix(".so.tmp%d" % os.getpid())
        res = subprocess.run([nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs)],
                             capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stderr}")
        os.replace(tmp, LIB)
    build_host(force)
    return LIB


def main():
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-v", action="store_true", help="print registers / spills per kernel")
    a = ap.parse_args()
    print(build(a.force, a.verbose or a.ptxas_v, a.ptxas_v))


if __name__ == "__main__":
    main()
