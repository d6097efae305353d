"""Build libpmx_moe_b200.so (the C-ABI library of include/pmx_moe.h) in-tree
with nvcc for sm_100a.  `python -m ppl.pmx_b200.build` or `build()`."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import threading

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "libpmx_moe_b200.so")
HOST = os.path.join(PKG, "_host_calls.so")       # the regular case of some operators' host side (csrc/host_calls.cpp)
SOURCES = ["cabi.cu", "select.cu", "elementwise.cu", "gemm_simt.cu", "gemm_tcgen05.cu", "gemm_tcgen05_pair.cu", "combine_allreduce.cu", "attention.cu", "mlp_tcgen05.cu",
           "rotary.cu", "cache_rows.cu", "masked_attention.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or add it to PATH")


def _stale(target: str) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if target == LIB or f == "host_calls.cpp"]
    deps.append(os.path.join(PKG, "..", "..", "include", "pmx_moe.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def _built_for() -> str:
    """What the host calls are built for; the package uses them where it is the same."""
    import torch
    return f"torch {torch.__version__}, python {sys.version_info[0]}.{sys.version_info[1]}"


def _host_stale() -> bool:
    if _stale(HOST):
        return True
    try:
        with open(HOST, "rb") as f:
            return _built_for().encode() + b"\0" not in f.read()
    except ImportError:                      # no torch: the build says so
        return True


def _host_command() -> list:
    import sysconfig
    import torch
    from torch.utils import cpp_extension
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(_nvcc()))), "include")
    inc = [f"-I{d}" for d in (*cpp_extension.include_paths(), cuda, sysconfig.get_paths()["include"])]
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    return ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-w", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            f'-DPMX_BUILT_FOR="{_built_for()}"', *inc, os.path.join(CSRC, "host_calls.cpp"), "-o", HOST + ".tmp", f"-L{lib}", "-lc10",
            "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]


def _build_host() -> None:
    """The host calls need torch's and Python's headers.  The operators run without them, a few microseconds a call later:
    a failure is reported and leaves none behind, and does not keep the library from being built."""
    try:
        done = subprocess.run(_host_command(), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
        failure = f"exit status {done.returncode}\n{done.stdout}" if done.returncode else ""
        if not done.returncode:
            os.replace(HOST + ".tmp", HOST)
    except Exception as e:
        failure = f"{type(e).__name__}: {e}\n"
    if failure:
        sys.stderr.write(f"--- host_calls.cpp was not built\n{failure}\n")
        if os.path.exists(HOST):
            os.remove(HOST)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every .cu of csrc/ into one shared library, and the host calls beside it; returns the library's path."""
    host = threading.Thread(target=_build_host)
    if force or _host_stale():
        host.start()
    try:
        return _build_library(verbose) if force or _stale(LIB) else LIB
    finally:
        if host.ident is not None:
            host.join()


def _build_library(verbose: bool) -> str:
    nvcc = _nvcc()
    objs = []
    procs = []
    for src in SOURCES:
        obj = os.path.join(CSRC, src[:-3] + ".o")
        cmd = [nvcc, *ARCH, "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
               "-Xptxas", "-v" if verbose else "-warn-spills", "-c", os.path.join(CSRC, src), "-o", obj]
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
        objs.append(obj)
    failed = False
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0 or verbose:
            sys.stderr.write(f"--- nvcc {src}\n{out}\n")
        failed |= p.returncode != 0
    if failed:
        raise RuntimeError("nvcc failed")
    tmp = LIB + ".tmp"
    subprocess.check_call([nvcc, *ARCH, "-shared", "-o", tmp, *objs, "-lcuda" if False else "-lcudart_static",
                           "-Xlinker", "--no-as-needed", "-ldl", "-lrt", "-lpthread"])
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
