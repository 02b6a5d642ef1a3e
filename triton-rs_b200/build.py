"""Build recipe for libb200_kernels.so (nvcc, sm_100a only, in-tree).

    python triton-rs_b200/build.py [--force] [--verbose]

The shared object is written next to this file so that it travels with the source
tree; nothing is cached outside the tree.
"""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
LIB = HERE / "libb200_kernels.so"
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=default",
]


def sources():
    return sorted(CSRC.glob("*.cu"))


def _stale() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    deps = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + [HERE.parent / "include" / "b200_kernels.h", Path(__file__), HERE / "fastcall.py"]
    return any(d.stat().st_mtime > t for d in deps)


def _build_calls(obj_dir):
    """The compiled argument conversion of the Python mirror (optional: without it the mirror converts in Python)."""
    import importlib.util
    mods = []
    for name in ("_lib", "fastcall"):
        spec = importlib.util.spec_from_file_location(f"b200k_{name}", HERE / f"{name}.py")
        mods.append(importlib.util.module_from_spec(spec))
        spec.loader.exec_module(mods[-1])
    mods[1].build(mods[0].parse_header(), obj_dir)


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not _stale():
        return LIB
    nvcc = os.environ.get("NVCC", "nvcc")
    objs = []
    obj_dir = HERE / "build"
    obj_dir.mkdir(exist_ok=True)
    procs = []
    for src in sources():
        obj = obj_dir / (src.stem + ".o")
        objs.append(obj)
        cmd = [nvcc, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = False
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0 or verbose:
            sys.stderr.write(f"--- {src.name}\n{out}\n")
        failed |= p.returncode != 0
    if failed:
        raise RuntimeError("nvcc failed")
    _build_calls(obj_dir)
    link = [nvcc, "-shared", "-o", str(LIB), *map(str, objs), "-lcudart"]
    subprocess.run(link, check=True)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
