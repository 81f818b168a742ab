"""Build libbusfill.so in-tree with nvcc (sm_100a only).

    python -m busfill_b200.build            # build if sources changed
    python -m busfill_b200.build --force -v # rebuild, show ptxas resource usage
"""
from __future__ import annotations

import argparse
import concurrent.futures
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB_DIR = os.path.join(PKG, "lib")
OBJ_DIR = os.path.join(PKG, "lib", "obj")
LIB_PATH = os.path.join(LIB_DIR, "libbusfill.so")
SOURCES = ["busfill.cu", "kv4.cu"]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found; CUDA 12.8+ is required to build libbusfill.so")
    return cand


def _inputs():
    files = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh", ".h"))]
    files.append(os.path.join(INCLUDE, "busfill.h"))
    files.append(os.path.abspath(__file__))
    return files


def up_to_date() -> bool:
    if not os.path.exists(LIB_PATH):
        return False
    t = os.path.getmtime(LIB_PATH)
    return all(os.path.getmtime(f) <= t for f in _inputs())


def _object_up_to_date(obj: str) -> bool:
    if not (os.path.exists(obj) and os.path.exists(obj + ".d")):
        return False
    with open(obj + ".d") as f:
        deps = f.read().replace("\\\n", " ").split(":", 1)[1].split()
    t = os.path.getmtime(obj)
    return all(os.path.exists(d) and os.path.getmtime(d) <= t for d in [*deps, os.path.abspath(__file__)])


def _run(cmd) -> str:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + res.stdout + res.stderr)
    return res.stdout + res.stderr


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    tmp = LIB_PATH + ".tmp"
    base = [nvcc_path(), *ARCH_FLAGS, "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
            "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr",
            f"-I{INCLUDE}", f"-I{CSRC}", "-DBUSFILL_BUILD"]
    if verbose:
        base.insert(1, "-Xptxas=-v")
    # one object per source, compiled side by side; an object newer than
    # everything its source includes is kept
    os.makedirs(OBJ_DIR, exist_ok=True)
    objects, jobs = [], []
    for src in SOURCES:
        obj = os.path.join(OBJ_DIR, src + ".o")
        objects.append(obj)
        if force or not _object_up_to_date(obj):
            jobs.append([*base, "-MD", "-MF", obj + ".d", "-c", os.path.join(CSRC, src), "-o", obj])
    with concurrent.futures.ThreadPoolExecutor(max(1, len(jobs))) as pool:
        for text in pool.map(_run, jobs):
            if verbose:
                sys.stderr.write(text)
    _run([*base, "-shared", *objects, "-o", tmp])
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))


if __name__ == "__main__":
    main()
