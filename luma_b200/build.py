"""Build ``luma_b200/_lib/libluma_b200.so`` with nvcc for sm_100a, and the
module ``luma_b200/_grads_ext.so`` (lists of torch tensors for the gradient
operators) with g++ against the installed torch.

    python -m luma_b200.build [--debug]

The library statically links the CUDA runtime, so it only needs the driver
(libcuda) at run time; without torch it is built alone.  The module works with
the torch and the Python it was built for, and says so when it is imported by
others.  The build output stays in-tree next to the package.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SOURCES = [os.path.join(HERE, "csrc", f"luma_{name}.cu") for name in ("step", "peer", "grad")]
OUT = os.path.join(HERE, "_lib", "libluma_b200.so")
EXT_SOURCE = os.path.join(HERE, "csrc", "luma_torch.cpp")
EXT_OUT = os.path.join(HERE, "_grads_ext.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC,-O2",
    "-shared",
]


def nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def build(verbose: bool = False, extra: list[str] | None = None) -> str:
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    cmd = [nvcc(), *NVCC_FLAGS, "-I", os.path.join(ROOT, "include"), *(extra or []),
           "-o", OUT + ".tmp", *SOURCES]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    os.replace(OUT + ".tmp", OUT)
    try:
        import torch  # noqa: F401
    except ImportError:
        print("no torch here: the library alone is built, without the module for its tensors")
    else:
        build_ext(verbose)
    return OUT


def build_ext(verbose: bool = False) -> str:
    """The torch-facing module; linked against the library and torch's own."""
    import torch
    from torch.utils import cpp_extension
    libs = cpp_extension.library_paths("cuda")
    cmd = [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared",
           "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DLUMA_TORCH_VERSION="{torch.__version__}"',
           "-I", os.path.join(ROOT, "include"),
           *(f"-isystem{p}" for p in cpp_extension.include_paths("cuda")),
           f"-isystem{sysconfig.get_paths()['include']}", EXT_SOURCE, "-o", EXT_OUT + ".tmp",
           "-L", os.path.dirname(OUT), "-lluma_b200", *(f"-L{p}" for p in libs),
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda",
           "-Wl,-rpath,$ORIGIN/_lib", *(f"-Wl,-rpath,{p}" for p in libs[:1])]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    os.replace(EXT_OUT + ".tmp", EXT_OUT)
    return EXT_OUT


def _older(out: str, deps: list[str]) -> bool:
    return not os.path.exists(out) or any(os.path.getmtime(s) > os.path.getmtime(out) for s in deps)


def is_stale() -> bool:
    header = os.path.join(ROOT, "include", "luma_b200.h")
    if _older(OUT, [*SOURCES, header, os.path.join(HERE, "csrc", "luma_internal.h")]):
        return True
    try:
        import torch  # noqa: F401
    except ImportError:
        return False  # the library is all there can be
    if _older(EXT_OUT, [EXT_SOURCE, header]):
        return True
    try:
        from luma_b200 import _grads_ext  # noqa: F401
    except ImportError:  # built for another torch, Python or library
        return True
    return False


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
