"""Build recipe for the in-tree CUDA library ``lmpool_b200/_kvx.so``.

The library is compiled with nvcc for sm_100a only (B200) and links the CUDA
runtime statically, so it needs nothing from PyTorch and loads on a machine
without a GPU (driver entry points are resolved at first use). Python reaches
it through ctypes (``lmpool_b200/_capi.py``); the C ABI is ``include/kvx.h``.

Usage: ``python -m lmpool_b200._build [--verbose]``.
"""
from __future__ import annotations

import argparse
import os
import re
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_ROOT = PKG_DIR.parent
SOURCES = [PKG_DIR / "csrc" / name for name in ("kvx.cu", "kvx_q4.cu", "kvx_attn.cu", "kvx_attn_split.cu", "kvx_attn_tile.cu")]
HEADERS = [REPO_ROOT / "include" / "kvx.h"] + [
    PKG_DIR / "csrc" / name for name in ("kvx_device.cuh", "kvx_host.h", "kvx_attn.cuh")]
OUTPUT = PKG_DIR / "_kvx.so"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3",
    "-std=c++17",
    "-lineinfo",
    "-Xcompiler",
    "-fPIC,-O2",
    "--expt-relaxed-constexpr",
    "-Xptxas",
    "-v",
]
LINK_FLAGS = ["-shared", "-Xcompiler", "-fPIC,-O2", "-cudart", "static"]
# Registers a thread of the kernels whose warps pass registers on to each other (setmaxnreg): their shares add up to
# what the block was launched with, so a build with any other number must not leave here.
REGISTERS = {"attn_tile_kernel": 96}


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the KV data path needs the CUDA 12.9 toolchain to build")


def is_stale() -> bool:
    if not OUTPUT.exists():
        return True
    out_m = OUTPUT.stat().st_mtime
    return any(p.stat().st_mtime > out_m for p in SOURCES + HEADERS)


def check_registers(ptxas_output: str) -> None:
    """Raises unless every kernel named in REGISTERS was built, with that many registers a thread."""
    found = {name: [] for name in REGISTERS}
    kernel = None
    for line in ptxas_output.splitlines():
        entry = re.search(r"Compiling entry function '(\w+)'", line)
        if entry:
            kernel = next((name for name in REGISTERS if name in entry.group(1)), None)
        used = re.search(r"Used (\d+) registers", line)
        if used and kernel:
            found[kernel].append(int(used.group(1)))
            kernel = None
    for name, counts in found.items():
        if not counts or any(n != REGISTERS[name] for n in counts):
            raise RuntimeError(f"{name} must be built with {REGISTERS[name]} registers a thread, this nvcc gave {counts}: "
                               f"its shares of setmaxnreg have to be set anew")


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> Path:
    """Compile the library if a source is newer than the built file."""
    if not force and not is_stale():
        return OUTPUT
    tmp = OUTPUT.with_suffix(".so.tmp")

    def run(*args: str) -> str:
        cmd = [nvcc_path(), *ARCH_FLAGS, *args]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
        return res.stdout + res.stderr

    # A process per source, so that what ptxas says of one does not mix with another's.
    with tempfile.TemporaryDirectory() as folder, ThreadPoolExecutor() as pool:
        objects = [str(Path(folder) / f"{src.stem}.o") for src in SOURCES]
        include = ["-I", str(REPO_ROOT / "include"), "-I", str(PKG_DIR / "csrc")]
        output = "".join(pool.map(lambda src, obj: run(*NVCC_FLAGS, *include, "-c", "-o", obj, str(src)), SOURCES, objects))
        check_registers(output)
        output += run(*LINK_FLAGS, "-o", str(tmp), *objects)
    if ptxas_info:
        sys.stderr.write(output)
    os.replace(tmp, OUTPUT)
    return OUTPUT


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true", help="print registers/spills per kernel")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose, ptxas_info=args.ptxas_info))


if __name__ == "__main__":
    main()
