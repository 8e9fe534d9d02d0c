"""Build libcq_b200.so in-tree with nvcc for sm_100a (one translation unit: csrc/libcq.cu), and _decode.so, the host side
of the decode-side operators on top of it, with the host compiler against torch's headers.

    python -m comfy_quant_bench_b200.build [--verbose]

The CUDA runtime is linked statically, so the library depends only on the NVIDIA driver; it shares the
process's primary context (and therefore torch's device memory and streams) through the driver.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libcq_b200.so")
SOURCES = ["libcq.cu", "rotquant.cu", "gemm_sm100.cu", "gemm_pair.cu", "gemv.cu", "dit.cu", "w4a16.cu", "w4a16_tokens.cu", "w4a16_mid.cu", "w4a16_tc.cu", "paged_attention.cu",
           "kvpages.cu", "selftest.cu", "capi.cu", "capi_decode.cu", "noalloc.cu", "kernels.cuh", "decode_common.cuh",
           "cq_common.cuh"]
HEADER = os.path.join(ROOT, "include", "cq_b200.h")
BIND_SRC = os.path.join(SRC, "decode_bind.cpp")
BIND = os.path.join(HERE, "_decode.so")


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put /usr/local/cuda/bin on PATH)")


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def needs_build() -> bool:
    return _stale(LIB, [os.path.join(SRC, s) for s in SOURCES] + [HEADER])


def _run(cmd: list[str], target: str, verbose: bool) -> None:
    """Runs a compiler that writes ``target`` + ".tmp", which then takes the target's place."""
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({res.returncode})")
    os.replace(target + ".tmp", target)


def _build_bind(verbose: bool) -> None:
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    cuda = os.path.dirname(os.path.dirname(nvcc_path()))
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    includes = [*cpp_extension.include_paths(), os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    _run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-w",
          "-DTORCH_EXTENSION_NAME=_decode", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          *(x for i in includes for x in ("-isystem", i)), BIND_SRC, "-o", BIND + ".tmp", "-L" + HERE, "-l:libcq_b200.so",
          "-Wl,-rpath,$ORIGIN", "-L" + libs, "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_cuda"], BIND, verbose)


def build(verbose: bool = False, force: bool = False) -> str:
    if force or needs_build():
        _run([nvcc_path(), "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
              "--expt-relaxed-constexpr", "-shared", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
              "-Xptxas", "-v" if verbose else "-O3", "-o", LIB + ".tmp", os.path.join(SRC, "libcq.cu")], LIB, verbose)
    if force or _stale(BIND, [BIND_SRC, HEADER]):
        _build_bind(verbose)
    return LIB


if __name__ == "__main__":
    print(build(verbose="--verbose" in sys.argv, force=True))
