"""Build the in-tree CUDA library ``_lib/liboscar_b200.so`` for sm_100a.

    python -m oscar_b200.build        (or __graft_entry__.build())

Two translation units (the INT2 path and the 16-bit paged path), compiled side
by side with nvcc for ``arch=compute_100a,code=sm_100a`` only and linked into
one shared library that travels with the source tree.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
SRCS = [PKG / "csrc" / "oscar_b200.cu", PKG / "csrc" / "paged16.cu"]
OUT = PKG / "_lib" / "liboscar_b200.so"
HEADERS = sorted((PKG / "csrc").glob("*.cuh")) + [PKG / "csrc" / "host.h", PKG.parent / "include" / "oscar_b200.h"]

NVCC_FLAGS = [
    "-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo",
    "-Xcompiler", "-fPIC", "-Xptxas", "-warn-spills",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def up_to_date() -> bool:
    if not OUT.exists():
        return False
    t = OUT.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in [*SRCS, *HEADERS])


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd))
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    if "spill" in (res.stderr or "").lower() and verbose:
        print(res.stderr)


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and up_to_date():
        return OUT
    OUT.parent.mkdir(parents=True, exist_ok=True)
    tmp = OUT.with_suffix(".so.tmp")
    with tempfile.TemporaryDirectory() as work:
        objs = [Path(work) / f"{src.stem}.o" for src in SRCS]
        cmds = [[nvcc(), *NVCC_FLAGS, "-c", "-o", str(obj), str(src)] for src, obj in zip(SRCS, objs)]
        with ThreadPoolExecutor(len(cmds)) as pool:
            list(pool.map(lambda cmd: _run(cmd, verbose), cmds))
        _run([nvcc(), *NVCC_FLAGS, "-shared", "-o", str(tmp), *map(str, objs)], verbose)
    os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
