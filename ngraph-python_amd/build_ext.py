"""Build libngraph_hip.so (the gfx950 kernels + C ABI) in-tree with hipcc.

Usage: ``python build_ext.py`` or ``build_all()`` from Python.  hipcc
cross-compiles for gfx950 without a GPU present.  The library lands in
``ngraph_hip/lib/`` next to the ctypes loader that opens it.
"""
from __future__ import print_function
import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
LIB_DIR = os.path.join(HERE, "ngraph_hip", "lib")
LIB_PATH = os.path.join(LIB_DIR, "libngraph_hip.so")

# translation units of the library; the first owns the contexts and the fused kernels
SOURCES = ["ngraph_hip.hip", "ngh_embedding.hip", "ngh_block_norm.hip", "ngh_block_norm_f32.hip", "ngh_block_norm_f16.hip",
           "ngh_block_norm_bf16.hip", "ngh_adamw.hip"]

HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-shared",
    # packed-fp32 instruction forms are kept out of every kernel
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # a*b+c must round twice, as the NumPy statements of the CPU transformer do
    "-ffp-contract=off",
    "-fno-gpu-rdc", "-Wno-unused-command-line-argument",
]


def find_hipcc():
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        raise RuntimeError("hipcc not found; libngraph_hip.so cannot be built")
    return hipcc


def build_all(verbose=True):
    """Compile every HIP source (side by side) and link libngraph_hip.so; returns its path."""
    if not os.path.isdir(LIB_DIR):
        os.makedirs(LIB_DIR)
    hipcc = find_hipcc()
    flags = HIPCC_FLAGS + os.environ.get("NGH_EXTRA_HIPCC_FLAGS", "").split()
    objects = tempfile.mkdtemp(prefix="ngh_build_")

    def run(cmd):
        if verbose:
            print(" ".join(cmd))
        return subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, universal_newlines=True)

    def compile_one(name):
        return run([hipcc] + [f for f in flags if f != "-shared"] + ["-I", INCLUDE, "-I", CSRC, "-c", os.path.join(CSRC, name),
                                                                    "-o", os.path.join(objects, name + ".o")])
    try:
        with ThreadPoolExecutor(max_workers=len(SOURCES)) as pool:
            procs = list(pool.map(compile_one, SOURCES))
        if all(p.returncode == 0 for p in procs):
            procs.append(run([hipcc] + flags + [os.path.join(objects, name + ".o") for name in SOURCES] + ["-o", LIB_PATH + ".tmp"]))
    finally:
        shutil.rmtree(objects, ignore_errors=True)
    for proc in procs:
        if proc.returncode != 0:
            raise RuntimeError("hipcc failed:\n" + proc.stdout)
        out = "\n".join(l for l in proc.stdout.splitlines()
                        if "packed-fp32-ops" not in l and l.strip())
        if verbose and out:
            print(out)
    os.replace(LIB_PATH + ".tmp", LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build_all(verbose="-q" not in sys.argv))
