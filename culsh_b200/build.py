"""Build the CUDA library in-tree:  python -m culsh_b200.build

Compiles the .cu files of culsh_b200/csrc for sm_100a, each into an object under build/ that is made again when a file it includes
is newer, and links them into culsh_b200/libculsh_b200.so (nvcc cross-compiles without a GPU).  The library exposes only the C ABI declared in
include/culsh_b200.h and links cudart + curand + the CUDA driver stub (for the tensor-map
encoder used by the TMA loads).
"""
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
SRCS = [os.path.join(HERE, "csrc", f) for f in ("culsh_b200.cu", "ranking.cu")]
OBJECTS = os.path.join(os.path.dirname(HERE), "build")
OUT = os.path.join(HERE, "libculsh_b200.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
]


def _sources():
    d = os.path.join(HERE, "csrc")
    inc = os.path.join(os.path.dirname(HERE), "include")
    out = [os.path.join(d, f) for f in sorted(os.listdir(d))]
    out += [os.path.join(inc, f) for f in sorted(os.listdir(inc))]
    return out


def is_stale() -> bool:
    if not os.path.exists(OUT):
        return True
    t = os.path.getmtime(OUT)
    return any(os.path.getmtime(s) > t for s in _sources())


def _run(cmd, verbose):
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
    if verbose:
        print(res.stderr)


def _object(nvcc, src, force, verbose):
    """The object of a source file, compiled if one of the files that it was made from last time is newer."""
    obj = os.path.join(OBJECTS, os.path.basename(src) + ".o")
    dep = obj + ".d"
    if not force and os.path.exists(obj) and os.path.exists(dep):
        files = open(dep).read().replace("\\\n", " ").split(":", 1)[1].split()
        if all(os.path.exists(f) and os.path.getmtime(f) <= os.path.getmtime(obj) for f in files):
            return obj
    _run([nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-MD", "-MF", dep, "-c", src, "-o", obj], verbose)
    return obj


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not is_stale():
        return OUT
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found: cannot build libculsh_b200.so")
    os.makedirs(OBJECTS, exist_ok=True)
    with ThreadPoolExecutor() as pool:
        objects = list(pool.map(lambda src: _object(nvcc, src, force, verbose), SRCS))
    _run([nvcc] + NVCC_FLAGS + ["-shared"] + objects + ["-o", OUT, "-lcurand"], verbose)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
