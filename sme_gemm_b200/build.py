"""Builds the CUDA library in-tree: sme_gemm_b200/libsmeg_b200.so (sm_100a only).

    python -m sme_gemm_b200.build [--force] [--verbose]

nvcc cross-compiles without a GPU; the .so is git-ignored but travels with the
source tree to the machine that runs it.
"""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libsmeg_b200.so")
SOURCES = ["api.cu", "q4_gemv.cu", "q4_mma.cu", "gemv_direct.cu", "lowbit_gemv.cu", "lowbit_tc.cu", "lowbit_mma.cu", "lowbit_rows.cu", "gemm_tc.cu", "elementwise.cu", "attention.cu", "rotary.cu", "paged.cu", "prompt.cu", "transcode.cu", "tp_reduce.cu", "pack.cc"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
         "-Xcompiler", "-fPIC,-ffp-contract=off,-Wall", "--expt-relaxed-constexpr"]


def _deps():
    out = []
    for root in (CSRC, os.path.join(os.path.dirname(HERE), "include")):
        for f in os.listdir(root):
            if f.endswith((".h", ".cuh")):
                out.append(os.path.join(root, f))
    return out


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    hdr_time = max(os.path.getmtime(p) for p in _deps())
    objs, rebuilt = [], False
    procs = []
    for src in SOURCES:
        sp = os.path.join(CSRC, src)
        op = os.path.join(OBJ, src + ".o")
        objs.append(op)
        stale = force or not os.path.exists(op) or os.path.getmtime(op) < max(os.path.getmtime(sp), hdr_time)
        if stale:
            cmd = [NVCC, *FLAGS, "-c", sp, "-o", op]
            if src.endswith(".cc"):
                cmd.insert(1, "-x")
                cmd.insert(2, "cu")
            if verbose:
                cmd.insert(1, "-Xptxas")
                cmd.insert(2, "-v")
            procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
            rebuilt = True
    for src, p in procs:
        out, _ = p.communicate()
        if verbose or p.returncode:
            sys.stderr.write(out)
        if p.returncode:
            raise RuntimeError(f"nvcc failed on {src}")
    if rebuilt or not os.path.exists(LIB):
        cmd = [NVCC, "-shared", "-o", LIB, *objs, "-gencode", "arch=compute_100a,code=sm_100a", "-lpthread"]
        subprocess.check_call(cmd)
    build_binding(force, verbose)
    return LIB


def _binding_command(torch):
    import sysconfig

    out = os.path.join(HERE, "_binding" + sysconfig.get_config_var("EXT_SUFFIX"))
    root = os.path.dirname(torch.__file__)
    inc = [sysconfig.get_paths()["include"], os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")]
    libs = os.path.join(root, "lib")
    return out, ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
                 *[x for i in inc for x in ("-isystem", i)], os.path.join(CSRC, "binding.cc"), "-o", out, f"-L{libs}", f"-Wl,-rpath,{libs}", "-ltorch_python", "-ltorch_cpu",
                 "-lc10", "-lc10_cuda"]


def build_binding(force: bool = False, verbose: bool = False) -> str | None:
    """The Python module behind paged.py (csrc/binding.cc): links against torch, takes the library's entry points by address.  It belongs to one torch:
    another version, place or ABI of it builds the module again.  None without torch, which the library does not need."""
    try:
        import torch                                           # (the one its headers belong to; it needs no GPU)
    except ImportError:
        sys.stderr.write("torch is not installed: the calls on packed batches (paged.py) are left out\n")
        return None
    out, cmd = _binding_command(torch)
    key = "\n".join([str(torch.__version__), *cmd]) + "\n"
    stamp = os.path.join(HERE, "_binding.stamp")
    sources = [os.path.join(CSRC, "binding.cc"), os.path.join(CSRC, "rows.h"), os.path.join(os.path.dirname(HERE), "include", "smeg_api.h")]
    if not force and os.path.exists(out) and os.path.exists(stamp) and os.path.getmtime(out) >= max(map(os.path.getmtime, sources)):
        with open(stamp) as f:
            if f.read() == key:
                return out
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if verbose or r.returncode:
        sys.stderr.write(r.stdout)
    if r.returncode:
        raise RuntimeError("g++ failed on binding.cc")
    with open(stamp, "w") as f:
        f.write(key)
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
