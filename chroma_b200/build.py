"""Build step: compile the sm_100a kernels and the C ABI into ``chroma_b200/libchroma_b200.so`` (in-tree), and the
binding of the operators on CUDA tensors into ``chroma_b200/_src/_tensors.so``.

nvcc cross-compiles without a GPU. The library links the CUDA runtime statically so it loads wherever the driver
is present. The binding is built against the installed Torch, and left out where there is none with CUDA; nothing but those
operators needs it.
"""

from __future__ import annotations

import importlib.util
import os
import runpy
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
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f'-DBUILT_FOR="{built_for()}"',
            str(TENSORS_SOURCE), "-o", str(target),
            "-I", sysconfig.get_paths()["include"], "-isystem", str(home / "include"), "-isystem",
            str(cuda / "include"), "-L", str(home / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]


def built_for() -> str | None:
    """The Torch and the Python that a binding built now is for; None without a Torch that has CUDA. Torch is not imported."""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.submodule_search_locations:
        return None
    version = runpy.run_path(str(Path(spec.submodule_search_locations[0]) / "version.py"))
    if not version.get("cuda"):
        return None
    return f"torch {version['__version__']}, {sysconfig.get_config_var('SOABI')}"


def stale(target: Path = TARGET, depends: list[Path] = DEPENDS) -> bool:
    if not target.exists():
        return True
    built = target.stat().st_mtime
    return any(p.stat().st_mtime > built for p in depends)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Builds what is not up to date. The library needs no Torch, and is in place whatever becomes of the binding."""
    jobs = []  # every command is put together before a compiler starts
    if force or stale(TARGET, DEPENDS):
        jobs.append((TARGET, TARGET.with_suffix(".so.tmp"), command(TARGET.with_suffix(".so.tmp"))))
    tag = built_for()
    if tag is None:
        if verbose:
            print("no Torch with CUDA: the binding of the operators on its tensors is left out", file=sys.stderr)
    elif force or stale(TENSORS, [TENSORS_SOURCE, *DEPENDS[-1:]]) or tag.encode() not in TENSORS.read_bytes():
        jobs.append((TENSORS, TENSORS.with_suffix(".so.tmp"), tensors_command(TENSORS.with_suffix(".so.tmp"))))
    running, failures = [], []
    for target, tmp, args in jobs:
        try:
            running.append((target, tmp, args, subprocess.Popen(args, stderr=subprocess.PIPE, text=True)))
        except OSError as error:
            failures.append(f"{Path(args[0]).name} failed:\n{error}")
    for target, tmp, args, process in running:
        _, messages = process.communicate()
        if process.returncode:
            failures.append(f"{Path(args[0]).name} failed:\n{messages}")
            tmp.unlink(missing_ok=True)
            continue
        if verbose and messages:
            print(messages, file=sys.stderr)
        os.replace(tmp, target)
    if failures:
        raise RuntimeError("\n".join(failures))
    return TARGET


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
