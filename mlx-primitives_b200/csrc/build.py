"""Build libmlxp_attn.so in-tree for sm_100a with nvcc (no torch extension machinery).

    python mlx-primitives_b200/csrc/build.py [--force] [--debug]

The library lands next to the Python package (mlx_primitives/libmlxp_attn.so) so that it
travels with the source tree; the Python shim loads it from there (or from $MLXP_LIB).  Beside it
goes _host.so, the C++ half of the shim (host_calls.cpp, built with g++ against torch's headers).
"""

from __future__ import annotations

import argparse
import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

CSRC = Path(__file__).resolve().parent
PKG_ROOT = CSRC.parent
INCLUDE = PKG_ROOT.parent / "include"
OUT = PKG_ROOT / "mlx_primitives" / "libmlxp_attn.so"
SOURCES = [CSRC / "mlxp_attn.cu", CSRC / "mlxp_cache.cu", CSRC / "mlxp_quant.cu",
           CSRC / "mlxp_quant_rows.cu"]
HOST_SOURCE = CSRC / "host_calls.cpp"
HOST_OUT = PKG_ROOT / "mlx_primitives" / "_host.so"
DEPS = SOURCES + [HOST_SOURCE] + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [INCLUDE / "mlxp_attn.h"]
OBJ = CSRC / "_build"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found (set $NVCC)")


def commands(debug: bool = False, verbose_ptxas: bool = False) -> tuple[list[list[str]], list[str]]:
    """The compile command of every source (they run in parallel) and the link command."""
    nvcc = nvcc_path()
    flags = [*ARCH, "-std=c++17", "-O3", "-lineinfo", "-Xcompiler", "-fPIC", "-cudart", "shared",
             "-I", str(INCLUDE)]
    if debug:
        flags += ["-DMLXP_DEBUG_CHECKS=1"]
    if verbose_ptxas:
        flags += ["-Xptxas", "-v"]
    objects = [OBJ / (s.stem + ".o") for s in SOURCES]
    compiles = [[nvcc, *flags, "-c", str(s), "-o", str(o)] for s, o in zip(SOURCES, objects)]
    link = [nvcc, *ARCH, "-shared", "-cudart", "shared",
            "-Xlinker", "-rpath,/usr/local/cuda/lib64", "-o", str(OUT), "-ldl",
            *map(str, objects)]
    return compiles, link


def host_command() -> list[str]:
    import torch

    root = Path(torch.__file__).resolve().parent
    return ["g++", "-O2", "-std=c++17", "-shared", "-fPIC",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            "-isystem", str(root / "include"),
            "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"),
            "-isystem", sysconfig.get_paths()["include"],
            "-isystem", str(Path(nvcc_path()).resolve().parent.parent / "include"),
            "-o", str(HOST_OUT), str(HOST_SOURCE),
            "-L", str(root / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python",
            f"-Wl,-rpath,{root / 'lib'}"]


def up_to_date() -> bool:
    if not OUT.exists() or not HOST_OUT.exists():
        return False
    t = min(OUT.stat().st_mtime, HOST_OUT.stat().st_mtime)
    return all(d.stat().st_mtime <= t for d in DEPS if d.exists())


def build(force: bool = False, debug: bool = False, verbose_ptxas: bool = False) -> Path:
    if not force and not debug and not verbose_ptxas and up_to_date():
        return OUT
    compiles, link = commands(debug=debug, verbose_ptxas=verbose_ptxas)
    OBJ.mkdir(exist_ok=True)

    def run(cmd):
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("compiler failed:\n" + " ".join(cmd) + "\n" + res.stdout + res.stderr)
        if verbose_ptxas:
            sys.stderr.write(res.stderr)

    with concurrent.futures.ThreadPoolExecutor() as pool:
        list(pool.map(run, [*compiles, host_command()]))
    run(link)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--debug", action="store_true")
    ap.add_argument("--ptxas-v", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, debug=a.debug, verbose_ptxas=a.ptxas_v))
