"""Build the sm_100a C-ABI library in-tree, attention_lab_b200/libattention_lab_b200.so, and the Python binding of its
8-bit cache operators, attention_lab_b200/_q8_bind.so (C++ against the installed torch, linked to the library).

    python -m attention_lab_b200.build [--verbose]

One nvcc compilation per csrc/*.cu (al_capi.cu: the sparse-decode path, al_q8.cu: the 8-bit cache; each includes its
kernel headers), run side by side, then one link; static CUDA runtime, position independent code. An object is compiled
again when its source, a header or this file is newer, or when its compiler line, torch or the Python ABI is another than
it was built with (kept beside it, and for the whole in _built.stamp). `--verbose` adds `-Xptxas -v` (registers, spills and shared memory per kernel).
"""
from __future__ import annotations

import argparse
import importlib.metadata
import importlib.util
import json
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
SRC = PKG / "csrc"
LIB = PKG / "libattention_lab_b200.so"
BIND = PKG / "_q8_bind.so"
OBJ = PKG / "_build"
STAMP = PKG / "_built.stamp"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[Path]:
    return [*sorted(f for pattern in ("*.cu", "*.cpp", "*.cuh", "*.h") for f in SRC.glob(pattern)),
            PKG.parent / "include" / "attention_lab_b200.h", PKG / "build.py"]


def made_with(commands) -> str:
    """What built files depend on besides their sources, wherever the tree lies."""
    return json.dumps({"torch": importlib.metadata.version("torch"), "abi": sysconfig.get_config_var("SOABI"),
                       "commands": commands}, indent=0).replace(str(PKG.parent), ".")


def stamp() -> str:
    return made_with([command(OBJ / (src.stem + ".o")) for src, command in compilations().items()]
                     + [link_library([]), link_bind(OBJ / "bind_q8.o")])


def up_to_date() -> bool:
    return (all(out.exists() and all(out.stat().st_mtime >= s.stat().st_mtime for s in sources()) for out in (LIB, BIND))
            and STAMP.exists() and STAMP.read_text() == stamp())


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


def bind_command(obj: Path) -> list[str]:
    """The compiler line of the binding's object (no torch import: its headers are found by location)."""
    torch_dir = Path(importlib.util.find_spec("torch").origin).parent
    cuda = Path(nvcc()).resolve().parents[1]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-D_GLIBCXX_USE_CXX11_ABI=1", "-I", str(torch_dir / "include"),
            "-I", sysconfig.get_paths()["include"], "-I", str(cuda / "include"), "-c", str(SRC / "bind_q8.cpp"),
            "-o", str(obj) + ".tmp"]


def link_bind(obj: Path) -> list[str]:
    torch_lib = Path(importlib.util.find_spec("torch").origin).parent / "lib"
    return ["g++", "-shared", str(obj), "-L", str(PKG), "-l:" + LIB.name, "-Wl,-rpath,$ORIGIN", "-L", str(torch_lib),
            "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", "-o", str(BIND) + ".tmp"]


def compilations() -> dict:
    """Source -> the compiler line that makes its object."""
    flags = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
             "-I", str(PKG.parent / "include")]
    lines = {src: lambda obj, src=src: [*flags, "-c", str(src), "-o", str(obj) + ".tmp"] for src in sorted(SRC.glob("*.cu"))}
    lines[SRC / "bind_q8.cpp"] = bind_command
    return lines


def link_library(objects) -> list[str]:
    return [nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", "-cudart", "static", *objects, "-o", str(LIB) + ".tmp"]


def build(verbose: bool = False, force: bool = False) -> Path:
    if up_to_date() and not force:
        return LIB
    OBJ.mkdir(exist_ok=True)
    jobs, objects = [], []
    for src, command in compilations().items():
        obj = OBJ / (src.stem + ".o")
        if src.suffix == ".cu":
            objects.append(str(obj))
        line = command(obj)
        made, note = made_with(line), obj.with_suffix(".made")
        if not force and obj.exists() and note.exists() and note.read_text() == made and all(
                obj.stat().st_mtime >= f.stat().st_mtime for f in included(src) | {Path(__file__).resolve()}):
            continue
        if verbose and src.suffix == ".cu":
            line.insert(1, "-Xptxas=-v")
        jobs.append((obj, note, made, subprocess.Popen(line, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = False
    for obj, note, made, job in jobs:
        out = job.communicate()[0]
        if job.returncode != 0 or verbose:
            sys.stderr.write(out)
        if job.returncode != 0:
            failed = True
        else:
            os.replace(str(obj) + ".tmp", obj)
            note.write_text(made)
    if failed:
        raise RuntimeError("compilation failed")
    for out, command in ((LIB, link_library(objects)), (BIND, link_bind(OBJ / "bind_q8.o"))):
        res = subprocess.run(command, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError(f"linking {out.name} failed with exit code {res.returncode}")
        os.replace(str(out) + ".tmp", out)
    STAMP.write_text(stamp())
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    print(build(verbose=a.verbose, force=a.force))
