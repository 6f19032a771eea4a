"""Build ``librapidalign_b200.so`` in-tree for sm_100a.

    python -m rapidalign_b200.build [--verbose]

One nvcc run for each source of ``csrc`` (objects under ``_build``, rebuilt
when a source or header is newer), all at once, then a link; the CUDA runtime
is linked statically so the library has no dependency beyond the driver.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "librapidalign_b200.so")
SOURCES = [os.path.join(CSRC, f) for f in ("ra_capi.cu", "ra_ce.cu", "ra_attn.cu")]
OBJ_DIR = os.path.join(HERE, "_build")
HEADERS = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))] + [
    os.path.join(HERE, os.pardir, "include", "rapidalign_b200.h")]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
]


def nvcc_path() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def up_to_date() -> bool:
    if not os.path.exists(OUT):
        return False
    t = os.path.getmtime(OUT)
    return all(os.path.getmtime(f) <= t for f in SOURCES + HEADERS + [__file__])


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return OUT
    os.makedirs(OBJ_DIR, exist_ok=True)
    newest = max(os.path.getmtime(f) for f in HEADERS + [__file__])
    objs, runs = [], []
    for src in SOURCES:
        obj = os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if not force and not verbose and os.path.exists(obj) and \
                os.path.getmtime(obj) > max(newest, os.path.getmtime(src)):
            continue
        part = obj + f".tmp{os.getpid()}"
        cmd = [nvcc_path(), *NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else []), "-c", "-o", part,
               src]
        runs.append((part, obj, subprocess.Popen(cmd, stdout=subprocess.PIPE,
                                                 stderr=subprocess.STDOUT, text=True)))
    said = [(part, obj, p.communicate()[0], p.returncode) for part, obj, p in runs]
    for part, obj, text, rc in said:
        if rc != 0:
            raise RuntimeError("nvcc failed:\n" + text)
        if verbose:
            sys.stderr.write(text)
        os.replace(part, obj)
    tmp = OUT + f".tmp{os.getpid()}"
    res = subprocess.run([nvcc_path(), *NVCC_FLAGS, "-shared", "-o", tmp, *objs],
                         capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
    os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
