"""Build the sm_100a C-ABI library in-tree: attention_lab_b200/libattention_lab_b200.so.

    python -m attention_lab_b200.build [--verbose]

One nvcc compilation per csrc/*.cu (al_capi.cu: the sparse-decode path, al_q8.cu: the 8-bit cache; each includes its
kernel headers), run side by side, then one link; static CUDA runtime, position independent code. An object is compiled
again when its source, a header or this file is newer. `--verbose` adds `-Xptxas -v` (registers, spills and shared memory per kernel).
"""
from __future__ import annotations

import argparse
import os
import re
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
SRC = PKG / "csrc"
LIB = PKG / "libattention_lab_b200.so"
OBJ = PKG / "_build"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[Path]:
    return sorted(SRC.glob("*.cu")) + sorted(SRC.glob("*.cuh")) + sorted(SRC.glob("*.h")) + [PKG.parent / "include" / "attention_lab_b200.h"]


def up_to_date() -> bool:
    return LIB.exists() and all(LIB.stat().st_mtime >= s.stat().st_mtime for s in sources())


def included(src: Path) -> set[Path]:
    """The source and every file of this tree it includes, directly or not."""
    seen, todo = set(), [src]
    while todo:
        f = todo.pop()
        if f in seen:
            continue
        seen.add(f)
        for name in re.findall(r'^\s*#include "([^"]+)"', f.read_text(), flags=re.M):
            inc = (f.parent / name).resolve()
            if inc.exists():
                todo.append(inc)
    return seen


def build(verbose: bool = False, force: bool = False) -> Path:
    if up_to_date() and not force:
        return LIB
    OBJ.mkdir(exist_ok=True)
    flags = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
             "-I", str(PKG.parent / "include")]
    if verbose:
        flags.insert(1, "-Xptxas=-v")
    jobs, objects = [], []
    for src in sorted(SRC.glob("*.cu")):
        obj = OBJ / (src.stem + ".o")
        objects.append(str(obj))
        if not force and obj.exists() and all(obj.stat().st_mtime >= f.stat().st_mtime
                                              for f in included(src) | {Path(__file__).resolve()}):
            continue
        jobs.append((obj, subprocess.Popen([*flags, "-c", str(src), "-o", str(obj) + ".tmp"], stdout=subprocess.PIPE,
                                           stderr=subprocess.STDOUT, text=True)))
    failed = False
    for obj, job in jobs:
        out = job.communicate()[0]
        if job.returncode != 0 or verbose:
            sys.stderr.write(out)
        if job.returncode != 0:
            failed = True
        else:
            os.replace(str(obj) + ".tmp", obj)
    if failed:
        raise RuntimeError("nvcc failed")
    res = subprocess.run([nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", "-cudart", "static", *objects,
                          "-o", str(LIB) + ".tmp"], capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"linking failed with exit code {res.returncode}")
    os.replace(str(LIB) + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    print(build(verbose=a.verbose, force=a.force))
