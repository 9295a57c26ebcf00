"""Build recipe for the in-tree sm_100a libraries.

``python -m decode_opt_b200.build`` compiles the library's sources in ``csrc/``
(``SOURCES``: the GEMM and its C ABI, probes, quantiser, and the attention
operators) into ``decode_opt_b200/libdecode_gemm_b200.so`` for ``sm_100a``
only, the files side by side.  The library links
the CUDA runtime statically and resolves ``cuTensorMapEncodeTiled``
through the runtime's driver entry-point query, so it loads on hosts without a
GPU (the CPU test suite checks its exported symbols there).

``csrc/dg_torch.cpp`` becomes ``decode_opt_b200/_host.so``, the extension
module through which ``attention.py`` makes the attention operators' calls
(host code against torch's C++ headers; it is handed the library's entry
points and links no CUDA code of its own).

It then compiles ``tests/cpp/dg_drop_in_check.cu`` against the C++ headers
(``include/decode_gemm.cuh``, ``include/weight_prepack.cuh``) and the
library into ``decode_opt_b200/dg_drop_in_check``, the program the GPU tests
run to check the C++ interface, and ``csrc/dg_cublaslt_fp8.cu`` into
``decode_opt_b200/dg_cublaslt_fp8``, the cuBLASLt FP8 baseline bench.py runs
in its own process (linked to the CUDA toolkit's cuBLASLt, which declares the
128-block scale modes; torch's bundled cuBLAS is never loaded beside it).
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB_NAME = "libdecode_gemm_b200.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
HOST_SRC = os.path.join(CSRC, "dg_torch.cpp")
HOST_LIB = os.path.join(HERE, "_host.so")
DROP_IN_SRC = os.path.join(ROOT, "tests", "cpp", "dg_drop_in_check.cu")
DROP_IN_BIN = os.path.join(HERE, "dg_drop_in_check")
CUBLASLT_SRC = os.path.join(CSRC, "dg_cublaslt_fp8.cu")
CUBLASLT_BIN = os.path.join(HERE, "dg_cublaslt_fp8")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
SOURCES = ("dg_capi.cu", "dg_probe.cu", "dg_quant.cu", "dg_block_tables.cu", "dg_rotary.cu", "dg_attention.cu")


def nvcc() -> str:
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = os.path.join(cuda_home, "bin", "nvcc")
    return cand if os.path.exists(cand) else (shutil.which("nvcc") or "nvcc")


def _sources():
    """What the nvcc-built programs are made of (the extension module's source
    is host code for torch's headers, and none of theirs)."""
    return [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f != os.path.basename(HOST_SRC)] + [
        os.path.join(INCLUDE, f) for f in sorted(os.listdir(INCLUDE))]


def needs_build(target: str = LIB_PATH, extra=()) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in list(_sources()) + list(extra))


def build(verbose: bool = False, ptxas_verbose: bool = False, force: bool = False) -> str:
    lib = build_cuda(verbose, ptxas_verbose, force)
    build_host(verbose, force)
    build_drop_in_check(verbose, force)
    build_cublaslt_bench(verbose, force)
    return lib


def host_built_for() -> str:
    """What the extension module is compiled against, as it says itself
    (``_host.built_for``)."""
    import torch
    python = f"{sys.version_info[0]}.{sys.version_info[1]}"
    return f"decode_opt_b200 host extension for torch {torch.__version__}, Python {python}"


def host_needs_build() -> bool:
    header = os.path.join(INCLUDE, "decode_attention_b200.h")
    if not os.path.exists(HOST_LIB) or \
            os.path.getmtime(HOST_LIB) <= max(os.path.getmtime(HOST_SRC), os.path.getmtime(header)):
        return True
    with open(HOST_LIB, "rb") as f:
        return host_built_for().encode() + b"\0" not in f.read()


def build_host(verbose: bool = False, force: bool = False) -> str:
    """The extension module of the attention operators' calls."""
    if not force and not host_needs_build():
        return HOST_LIB
    if os.path.exists(HOST_LIB):
        os.remove(HOST_LIB)          # of other sources: it would pass structs of another layout
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    flags = [f"-I{os.path.join(root, 'include')}", f"-I{os.path.join(root, 'include', 'torch', 'csrc', 'api', 'include')}",
             f"-I{sysconfig.get_paths()['include']}", f"-I{os.path.join(cuda_lib_dir(), '..', 'include')}", f"-I{INCLUDE}"]
    cmd = [os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DDG_BUILT_FOR="{host_built_for()}"', *flags, HOST_SRC, "-o",
           HOST_LIB + ".tmp", "-L", os.path.join(root, "lib"), "-L", cuda_lib_dir(), "-lc10", "-lc10_cuda", "-ltorch",
           "-ltorch_cpu", "-ltorch_python", "-lcudart"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(HOST_LIB + ".tmp", HOST_LIB)
    return HOST_LIB


def build_library(verbose: bool = False, ptxas_verbose: bool = False, force: bool = False) -> str:
    """The C library, which needs no torch; then the extension module, without
    which attention.py says so when it is first used."""
    lib = build_cuda(verbose, ptxas_verbose, force)
    try:
        build_host(verbose, force)
    except (ImportError, OSError, subprocess.CalledProcessError) as e:
        print(f"{HOST_LIB} was not built: {e}", file=sys.stderr)
    return lib


def cuda_lib_dir() -> str:
    return os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "lib64")


def build_cublaslt_bench(verbose: bool = False, force: bool = False) -> str:
    """The cuBLASLt FP8 baseline program (block-scaled and per-tensor)."""
    if not force and os.path.exists(CUBLASLT_BIN) and os.path.getmtime(CUBLASLT_BIN) > os.path.getmtime(CUBLASLT_SRC):
        return CUBLASLT_BIN
    libdir = cuda_lib_dir()
    cmd = [nvcc(), "-std=c++17", "-O3", *ARCH_FLAGS, CUBLASLT_SRC, "-o", CUBLASLT_BIN + ".tmp", "-L", libdir,
           "-lcublasLt", "-Xlinker", f"-rpath,{libdir}"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(CUBLASLT_BIN + ".tmp", CUBLASLT_BIN)
    return CUBLASLT_BIN


def build_drop_in_check(verbose: bool = False, force: bool = False) -> str:
    """The C++-interface check program, linked to the in-tree library (found
    next to it at run time)."""
    if not force and not needs_build(DROP_IN_BIN, (DROP_IN_SRC, LIB_PATH)):
        return DROP_IN_BIN
    cmd = [nvcc(), "-std=c++17", "-O3", "-lineinfo", *ARCH_FLAGS, "-I", INCLUDE, "-I", CSRC, DROP_IN_SRC,
           "-o", DROP_IN_BIN + ".tmp", "-L", HERE, "-ldecode_gemm_b200", "-Xlinker", "-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(DROP_IN_BIN + ".tmp", DROP_IN_BIN)
    return DROP_IN_BIN


def build_cuda(verbose: bool = False, ptxas_verbose: bool = False, force: bool = False) -> str:
    """The C library alone."""
    if not force and not needs_build(LIB_PATH):
        return LIB_PATH
    cmd = [nvcc(), "-std=c++17", "-O3", "-lineinfo", *ARCH_FLAGS,
           "-Xcompiler", "-fPIC", "-shared", "-cudart", "static", "--threads", "0",
           "-I", CSRC, "-I", INCLUDE,
           *[os.path.join(CSRC, f) for f in SOURCES], "-o", LIB_PATH + ".tmp"]
    if ptxas_verbose:
        cmd[1:1] = ["-Xptxas", "-v"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(LIB_PATH + ".tmp", LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    build(verbose=True, ptxas_verbose="-v" in sys.argv, force="-f" in sys.argv)
