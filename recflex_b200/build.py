"""Build librecflex_b200.so in-tree with nvcc for sm_100a.

Run `python -m recflex_b200.build` (or call `build()`).  The fused kernel is
compiled once per CTAs-per-SM occupancy; those translation units are
independent and build in parallel.  Objects land in `recflex_b200/build/`, the
library beside the package as `recflex_b200/librecflex_b200.so`.
"""
from __future__ import annotations

import concurrent.futures
import contextlib
import hashlib
import os
import re
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
BUILD_DIR = os.path.join(PKG_DIR, "build")
LIB_PATH = os.path.join(PKG_DIR, "librecflex_b200.so")
INCLUDE_DIR = os.path.join(os.path.dirname(PKG_DIR), "include")

NVCC_FLAGS = [
    "-O3",
    "-std=c++17",
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-Xcompiler",
    "-fPIC",
]


def _nvcc() -> str:
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found; the library cannot be built")
    return nvcc


_INCLUDE = re.compile(r'^\s*#\s*include\s+"([^"]+)"', re.M)


def _unit_digest(unit) -> str:
    """Digest of what an object is built from: its source, the headers that it includes by quotes, and the flags."""
    _, src, extra = unit
    h = hashlib.sha256(" ".join(NVCC_FLAGS + extra).encode())
    todo, seen = [os.path.join(CSRC, src)], set()
    while todo:
        path = os.path.normpath(todo.pop())
        if path in seen or not os.path.isfile(path):
            continue
        seen.add(path)
        with open(path, "rb") as f:
            text = f.read()
        h.update(os.path.basename(path).encode() + text)
        todo += [os.path.join(os.path.dirname(path), name) for name in sorted(_INCLUDE.findall(text.decode()))]
    return h.hexdigest()


def _units():
    """(object name, source, extra flags)"""
    units = [
        ("eb_capi.o", "eb_capi.cu", []),
        ("eb_launch.o", "eb_launch.cu", []),
        ("eb_noalloc.o", "eb_noalloc.cu", []),
        ("eb_warp.o", "eb_warp_inst.cu", []),
        ("eb_longbag.o", "eb_longbag_inst.cu", []),
        ("eb_rows.o", "eb_rows.cu", []),
        ("eb_linear.o", "eb_linear.cu", []),
        ("eb_linear_few.o", "eb_linear_few.cu", []),
    ]
    for occ in range(1, 9):
        units.append((f"eb_fused_occ{occ}.o", "eb_fused_inst.cu", [f"-DEB_OCC={occ}"]))
    return [u for u in units if os.path.exists(os.path.join(CSRC, u[1]))]


def _compile(unit, force: bool, verbose: bool) -> str:
    obj, src, extra = unit
    out = os.path.join(BUILD_DIR, obj)
    stamp, digest = out + ".sha256", _unit_digest(unit)
    if not force and os.path.exists(out) and _read(stamp) == digest:
        return digest
    cmd = [_nvcc(), *NVCC_FLAGS, *extra, "-I", INCLUDE_DIR, "-c", os.path.join(CSRC, src)]
    if verbose:
        cmd.insert(1, "-Xptxas")
        cmd.insert(2, "-v")
    res = _produce(cmd, out, stamp, digest, f"nvcc failed for {src} {extra}")
    if verbose:
        sys.stderr.write(res.stderr)
    return digest


def _produce(cmd, out: str, stamp: str, digest: str, failure: str):
    """Run `cmd -o out` and note in `stamp` what `out` was made of.

    The old note goes first and the new one comes last, and the output takes its place whole: wherever this ends, and
    beside another process that builds, there is no note of an output that is not the one it names."""
    fresh = f"{out}.{os.getpid()}.new"
    with contextlib.suppress(FileNotFoundError):
        os.remove(stamp)
    try:
        res = subprocess.run([*cmd, "-o", fresh], capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"{failure}:\n{res.stdout}\n{res.stderr}")
        os.replace(fresh, out)
    finally:
        with contextlib.suppress(FileNotFoundError):
            os.remove(fresh)
    with open(stamp, "w") as f:
        f.write(digest)
    return res


def _read(path: str) -> str:
    try:
        with open(path) as f:
            return f.read().strip()
    except FileNotFoundError:  # never there, or taken away just now by another process that builds
        return ""


def build(force: bool = False, verbose: bool = False, jobs: int | None = None) -> str:
    """Compile the units whose sources changed, link, and return the path of the shared library."""
    units = _units()
    stamp = os.path.join(BUILD_DIR, "sources.sha256")
    # checked before anything is written: several processes may ask for an up-to-date library at once
    digest = hashlib.sha256(" ".join(_unit_digest(u) for u in units).encode()).hexdigest()
    if not force and os.path.exists(LIB_PATH) and _read(stamp) == digest:
        return LIB_PATH
    os.makedirs(BUILD_DIR, exist_ok=True)
    jobs = jobs or min(len(units), os.cpu_count() or 1)
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as pool:
        list(pool.map(lambda u: _compile(u, force, verbose), units))
    objs = [os.path.join(BUILD_DIR, u[0]) for u in units]
    cmd = [_nvcc(), "-shared", "-gencode", "arch=compute_100a,code=sm_100a", *objs]
    _produce(cmd, LIB_PATH, stamp, digest, "link failed")
    return LIB_PATH


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(path)
