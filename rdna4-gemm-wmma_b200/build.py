"""Build libb2g_gemm.so in-tree with nvcc for sm_100a.

    python rdna4-gemm-wmma_b200/build.py [--verbose]

The library is plain nvcc output (static CUDA runtime, no framework dependency) so a C or
C++ caller can link or dlopen it directly; Python callers use b2g.py (ctypes).
"""
import argparse
import concurrent.futures
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libb2g_gemm.so")
SOURCES = ["b2g_api.cu", "b2g_shard.cu", "b2g_rows.cu", "b2g_q8.cu"]
HEADERS = ["ptx.cuh", "gemm_sm100.cuh", "sched.h", "errors.h", "plan.h", "host.h", "q8.cuh",
           "skinny_sm100.cuh"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-v",
]
LINK_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC", "-ldl"]
OBJ = os.path.join(HERE, "obj")  # one object and one ptxas log per source


def nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _newer(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def _deps(sources):
    return [os.path.join(CSRC, f) for f in sources + HEADERS] + [
        os.path.join(ROOT, "include", "b2g_gemm.h"), os.path.abspath(__file__)]


def stale():
    return _newer(LIB, _deps(SOURCES))


def _read_deps(path, src):
    """Files that a source was last compiled from, as the compiler listed them."""
    if not os.path.exists(path):
        return _deps([src])
    words = open(path).read().replace("\\\n", " ").split(":", 1)[1].split()
    return [w for w in words if w.startswith(ROOT)] + [os.path.abspath(__file__)]


def _compile(src, force, verbose):
    """Object file of one source, compiled unless it is up to date."""
    obj = os.path.join(OBJ, src + ".o")
    if not force and not _newer(obj, _read_deps(obj + ".d", src)):
        return obj
    cmd = [nvcc()] + NVCC_FLAGS + ["-I", os.path.join(ROOT, "include"), "-MD", "-MF",
                                   obj + ".d", "-c", "-o", obj + ".tmp", os.path.join(CSRC, src)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed compiling " + src)
    with open(obj + ".log", "w") as f:
        f.write(res.stderr)
    os.replace(obj + ".tmp", obj)
    return obj


def build(force=False, verbose=False):
    if not force and not stale():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    with concurrent.futures.ThreadPoolExecutor(len(SOURCES)) as pool:
        objs = list(pool.map(lambda s: _compile(s, force, verbose), SOURCES))
    res = subprocess.run([nvcc()] + LINK_FLAGS + ["-o", LIB + ".tmp"] + objs, capture_output=True,
                         text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed linking libb2g_gemm.so")
    os.replace(LIB + ".tmp", LIB)
    # keep the ptxas resource summary next to the build for inspection
    with open(os.path.join(HERE, "ptxas_resources.txt"), "w") as f:
        for o in objs:
            f.write("\n".join(l for l in open(o + ".log").read().splitlines() if "ptxas info" in l) + "\n")
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
