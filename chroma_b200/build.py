"""Build step: compile the sm_100a kernels and the C ABI into ``chroma_b200/libchroma_b200.so`` (in-tree), and the
binding of the operators on CUDA tensors into ``chroma_b200/_src/_tensors.so``.

nvcc cross-compiles without a GPU. The library links the CUDA runtime statically so it loads wherever the driver
is present. The binding is built against the installed Torch; nothing but those operators needs it.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
ROOT = PACKAGE.parent
SOURCES = [PACKAGE / "csrc" / "runtime.cu", PACKAGE / "csrc" / "graph.cu", PACKAGE / "csrc" / "ops.cu"]
DEPENDS = sorted((PACKAGE / "csrc").glob("*.cu*")) + [ROOT / "include" / "chroma_b200.h"]
TARGET = PACKAGE / "libchroma_b200.so"
TENSORS = PACKAGE / "_src" / "_tensors.so"
TENSORS_SOURCE = PACKAGE / "csrc" / "tensors.cpp"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    found = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists() and shutil.which(found) is None:
        raise RuntimeError("nvcc not found; set NVCC or add the CUDA toolkit to PATH")
    return found


def command(target: Path = TARGET) -> list[str]:
    return [nvcc(), "-O3", "-std=c++17", *ARCH, "-lineinfo", "-Xcompiler", "-fPIC", "-shared", "--cudart=static", "--threads", "0",
            "-I", str(ROOT / "include"), *map(str, SOURCES), "-o", str(target)]


def tensors_command(target: Path = TENSORS) -> list[str]:
    import torch

    home = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parents[1]
    return [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", str(TENSORS_SOURCE), "-o", str(target),
            "-I", sysconfig.get_paths()["include"], "-isystem", str(home / "include"), "-isystem",
            str(cuda / "include"), "-L", str(home / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]


def stale(target: Path = TARGET, depends: list[Path] = DEPENDS) -> bool:
    if not target.exists():
        return True
    built = target.stat().st_mtime
    return any(p.stat().st_mtime > built for p in depends)


def build(force: bool = False, verbose: bool = False) -> Path:
    jobs = []
    for target, depends, make in ((TARGET, DEPENDS, command), (TENSORS, [TENSORS_SOURCE, *DEPENDS[-1:]], tensors_command)):
        if force or stale(target, depends):
            tmp = target.with_suffix(".so.tmp")
            args = make(tmp)
            jobs.append((target, tmp, args[0], subprocess.Popen(args, stderr=subprocess.PIPE, text=True)))
    for target, tmp, compiler, process in jobs:
        _, messages = process.communicate()
        if process.returncode:
            raise RuntimeError(f"{Path(compiler).name} failed:\n{messages}")
        if verbose and messages:
            print(messages, file=sys.stderr)
        os.replace(tmp, target)
    return TARGET


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
