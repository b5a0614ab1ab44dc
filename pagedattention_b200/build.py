"""Build libpab200.so in-tree with nvcc for sm_100a.

    python -m pagedattention_b200.build [--verbose]

The shared library lands next to this file (pagedattention_b200/libpab200.so),
which is where ``pagedattention_b200._lib`` loads it from.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
LIB_PATH = PKG_DIR / "libpab200.so"
OBJ_DIR = PKG_DIR / "build"
SOURCES = [CSRC / "pab200.cu", CSRC / "int4_decode.cu", CSRC / "int4.cu", CSRC / "sparse.cu"]
HEADERS = [CSRC / "append.cuh", CSRC / "decode.cuh", CSRC / "int4.cuh", CSRC / "int4_decode.cuh",
           CSRC / "ptx.cuh", CSRC / "tokens.cuh", CSRC / "host.h", REPO_DIR / "include" / "pab200.h"]

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libpab200.so")
    return cand


def compile_command(src: Path, obj: Path, verbose_ptxas: bool = False) -> list[str]:
    cmd = [
        nvcc_path(), *ARCH_FLAGS, "-O3", "-lineinfo", "-std=c++17",
        "-Xcompiler", "-fPIC,-fvisibility=hidden",
        "-I", str(REPO_DIR / "include"), "-I", str(CSRC), "-c", str(src), "-o", str(obj),
    ]
    if verbose_ptxas:
        cmd += ["-Xptxas", "-v"]
    return cmd


def link_command(objs: list[Path], out: Path) -> list[str]:
    return [nvcc_path(), *ARCH_FLAGS, "-shared", "-o", str(out), *map(str, objs)]


def is_stale() -> bool:
    if not LIB_PATH.exists():
        return True
    t = LIB_PATH.stat().st_mtime
    return any(p.stat().st_mtime > t for p in SOURCES + HEADERS)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library if it is missing or older than its sources."""
    if not force and not is_stale():
        return LIB_PATH
    OBJ_DIR.mkdir(exist_ok=True)
    objs = [OBJ_DIR / (src.stem + ".o") for src in SOURCES]
    headers = max(p.stat().st_mtime for p in HEADERS)

    def run(cmd):
        res = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed ({res.returncode}): {' '.join(cmd)}")

    def compile_one(pair):
        src, obj = pair
        if (force or not obj.exists()
                or obj.stat().st_mtime < max(headers, src.stat().st_mtime)):
            part = obj.with_suffix(".o.tmp")
            run(compile_command(src, part, verbose_ptxas=verbose))
            os.replace(part, obj)

    with ThreadPoolExecutor(len(SOURCES)) as pool:
        list(pool.map(compile_one, zip(SOURCES, objs)))
    tmp = LIB_PATH.with_suffix(".so.tmp")
    run(link_command(objs, tmp))
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true", help="print ptxas register/spill report")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))


if __name__ == "__main__":
    main()
