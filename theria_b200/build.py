"""Build libtheria_sm100.so in-tree with nvcc (sm_100a only).

    python -m theria_b200.build [--verbose]

The library is three translation units (csrc/theria_sm100.cu, csrc/theria_lm.cu,
csrc/theria_ragged.cu) compiled side by side for ``arch=compute_100a,code=sm_100a``; nvcc
cross-compiles them on a machine without a GPU.  The output lands next to this
file so it travels with the source tree.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libtheria_sm100.so")
ROOT = os.path.dirname(HERE)
OBJ = os.path.join(HERE, "_build")
UNITS = ("theria_sm100", "theria_lm", "theria_ragged")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc():
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: cannot build libtheria_sm100.so")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC)
                  if f.endswith((".cu", ".cuh")))


def headers():
    inc = os.path.join(ROOT, "include")
    return [os.path.join(inc, h) for h in sorted(os.listdir(inc)) if h.endswith(".h")]


def _newer(out, deps):
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    return all(os.path.getmtime(p) <= t for p in deps if os.path.exists(p))


def _deps(unit):
    # the headers csrc/lm_* belong to theria_lm alone, csrc/ragged_* to theria_ragged
    def belongs(p):
        first = os.path.basename(p).split("_")[0]
        return first not in ("lm", "ragged") or unit == "theria_" + first
    cu = os.path.join(CSRC, unit + ".cu")
    deps = [p for p in sources() if p.endswith(".cuh") and belongs(p)]
    return [cu] + deps + headers() + [__file__]


def up_to_date():
    return _newer(LIB, sources() + headers() + [__file__])


def build(force: bool = False, verbose: bool = False, extra=()) -> str:
    if not force and up_to_date():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    nvcc = _nvcc()
    objs, jobs = [], []
    for unit in UNITS:
        obj = os.path.join(OBJ, unit + ".o")
        objs.append(obj)
        if not force and _newer(obj, _deps(unit)):
            continue
        cmd = [nvcc, *NVCC_FLAGS, *extra, "-I", os.path.join(ROOT, "include"), "-c",
               os.path.join(CSRC, unit + ".cu"), "-o", obj + ".tmp"]
        if verbose:
            print(" ".join(cmd), flush=True)
        jobs.append((cmd, obj, subprocess.Popen(cmd)))
    status = [p.wait() for _, _, p in jobs]  # all ended before any error is raised
    for (cmd, obj, _), rc in zip(jobs, status):
        if rc != 0:
            raise subprocess.CalledProcessError(rc, cmd)
        os.replace(obj + ".tmp", obj)
    link = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", *objs, "-o",
            LIB + ".tmp", "-lcuda"]
    if verbose:
        print(" ".join(link), flush=True)
    subprocess.run(link, check=True)
    os.replace(LIB + ".tmp", LIB)
    return LIB


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-v", action="store_true", help="print register/smem use")
    a = ap.parse_args()
    extra = ["-Xptxas", "-v"] if a.ptxas_v else []
    print(build(force=a.force or a.ptxas_v, verbose=a.verbose, extra=extra))


if __name__ == "__main__":
    sys.exit(main())
