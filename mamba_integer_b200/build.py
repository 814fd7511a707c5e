"""Build the sm_100a CUDA library ``libmi_b200.so`` in-tree.

The library is one nvcc translation unit (csrc/mi_b200_unity.cu) exposing the
C ABI declared in include/mi_b200.h.  It links the CUDA runtime statically, so
loading it needs no GPU; the driver is reached at the first CUDA call.

    python -m mamba_integer_b200.build
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
ROOT = os.path.dirname(HERE)
SO = os.path.join(HERE, "libmi_b200.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    # IEEE-exact float arithmetic: no contraction, IEEE div/sqrt, no flush-to-zero
    "-fmad=false", "-prec-div=true", "-prec-sqrt=true", "-ftz=false",
    "-Xcompiler", "-fPIC", "-shared",
]


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))


def needs_build() -> bool:
    if not os.path.exists(SO):
        return True
    t = os.path.getmtime(SO)
    deps = _sources() + [os.path.join(ROOT, "include", "mi_b200.h")]
    return any(os.path.getmtime(s) > t for s in deps)


BPE_SO = os.path.join(HERE, "libmi_bpe.so")
BPE_SRC = os.path.join(HERE, "tokenizer", "bpe.cpp")


def build_bpe(force: bool = False) -> str:
    """The host-side tokenizer library libmi_bpe.so (g++, C++17)."""
    deps = [BPE_SRC, os.path.join(HERE, "tokenizer", "unicode_classes.h"), os.path.join(ROOT, "include", "mi_bpe.h")]
    if not force and os.path.exists(BPE_SO) and all(os.path.getmtime(d) <= os.path.getmtime(BPE_SO) for d in deps):
        return BPE_SO
    cxx = shutil.which("g++") or "g++"
    subprocess.run([cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-o", BPE_SO + ".tmp", BPE_SRC], check=True)
    os.replace(BPE_SO + ".tmp", BPE_SO)
    return BPE_SO


TORCH_SO = os.path.join(HERE, "_mi_torch.so")
TORCH_SRC = os.path.join(CSRC, "torch_ops.cpp")
TORCH_STAMP = TORCH_SO + ".stamp"


def torch_stamp() -> str:
    """What _mi_torch.so is tied to beside its sources: another torch or Python than it was built for needs a new one."""
    import torch

    return "\n".join([torch.__version__, os.path.dirname(torch.__file__), str(int(torch._C._GLIBCXX_USE_CXX11_ABI)),
                      sys.version, sys.implementation.cache_tag]) + "\n"


def torch_needs_build() -> bool:
    deps = [TORCH_SRC, os.path.join(ROOT, "include", "mi_b200.h")]
    if not os.path.exists(TORCH_SO) or any(os.path.getmtime(d) > os.path.getmtime(TORCH_SO) for d in deps):
        return True
    try:
        with open(TORCH_STAMP) as f:
            return f.read() != torch_stamp()
    except OSError:
        return True


def build_torch(force: bool = False) -> str:
    """The float operators' calls from torch, _mi_torch.so (g++, C++17; no CUDA compiler)."""
    if not force and not torch_needs_build():
        return TORCH_SO
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cxx = shutil.which("g++") or "g++"
    cuda = os.path.dirname(os.path.dirname(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"))
    includes = [*cpp_extension.include_paths(), os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    subprocess.run([cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
                    "-DTORCH_EXTENSION_NAME=_mi_torch", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                    *[arg for path in includes for arg in ("-isystem", path)], "-o", TORCH_SO + ".tmp", TORCH_SRC,
                    "-L" + libs, "-Wl,-rpath," + libs, "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"],
                   check=True)
    if os.path.exists(TORCH_STAMP):
        os.remove(TORCH_STAMP)  # never an old stamp beside a new library
    os.replace(TORCH_SO + ".tmp", TORCH_SO)
    with open(TORCH_STAMP, "w") as f:
        f.write(torch_stamp())
    return TORCH_SO


def build(verbose: bool = False, force: bool = False) -> str:
    build_bpe(force=force)
    build_torch(force=force)
    if not force and not needs_build():
        return SO
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    cmd = [nvcc, *NVCC_FLAGS, "-o", SO + ".tmp", os.path.join(CSRC, "mi_b200_unity.cu")]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True, cwd=CSRC)
    os.replace(SO + ".tmp", SO)
    return SO


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force=True))
