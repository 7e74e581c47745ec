"""Ahead-of-time build of ``libb200nn.so`` (sm_100a only) and of ``b200_torch_calls.so``, the module that calls it with torch tensors.

``python build_native.py`` or ``build()`` compiles every ``csrc/*.cu`` with nvcc and
links one shared library next to the Python runtime package, where
``cuda_runtime.native`` loads it with ctypes.  nvcc cross-compiles without a GPU.
Objects are rebuilt only when their source (or a header) is newer.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import warnings
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

ROOT = Path(__file__).resolve().parent
CSRC = ROOT / "csrc"
OBJ_DIR = CSRC / "build"
LIB_PATH = ROOT / "cuda_runtime" / "libb200nn.so"
CALLS_PATH = ROOT / "cuda_runtime" / "b200_torch_calls.so"
INCLUDE = ROOT.parent / "include"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-I", str(INCLUDE),
]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; the b200nn library must be built with the CUDA 12.9 toolkit")
    return exe


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def build(force: bool = False, verbose: bool = False) -> Path:
    nvcc = _nvcc()
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    headers = list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    newest_header = max((h.stat().st_mtime for h in headers), default=0.0)
    flags = list(NVCC_FLAGS)

    def compile_one(src: Path) -> Path:
        obj = OBJ_DIR / (src.stem + ".o")
        if not force and obj.exists() and obj.stat().st_mtime > max(src.stat().st_mtime, newest_header):
            return obj
        cmd = [nvcc, *flags, "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
        return obj

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        objs = list(pool.map(compile_one, sources()))
    if force or not LIB_PATH.exists() or any(o.stat().st_mtime > LIB_PATH.stat().st_mtime for o in objs):
        cmd = [nvcc, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-cudart", "static",
               "-o", str(LIB_PATH), *map(str, objs)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    try:
        build_torch_calls(force, verbose)
    except (RuntimeError, ImportError, OSError) as exc:   # (the library serves callers without torch, too; calls with tensors raise until the module is there)
        warnings.warn(f"{CALLS_PATH.name} was not built: {exc}")
    return LIB_PATH


def build_torch_calls(force: bool = False, verbose: bool = False) -> Path:
    """``csrc/torch_calls.cpp`` against the headers of the torch that is installed.  Built again when its source, the library's header, the
    torch or the interpreter is another one than it was built with."""
    import sysconfig

    import torch

    from cuda_runtime import native

    src = CSRC / "torch_calls.cpp"
    built_for = native.torch_calls_built_for()
    if not force and CALLS_PATH.exists() and CALLS_PATH.stat().st_mtime > max(src.stat().st_mtime, (INCLUDE / "b200nn.h").stat().st_mtime) and \
            built_for.encode() in CALLS_PATH.read_bytes():
        return CALLS_PATH
    base = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parents[1]
    includes = [base / "include", base / "include" / "torch" / "csrc" / "api" / "include", sysconfig.get_paths()["include"], cuda / "include"]
    CALLS_PATH.unlink(missing_ok=True)   # (where it does not compile, what was there is not to be loaded)
    made = CALLS_PATH.with_suffix(f".{os.getpid()}.so")   # (nobody finds half of it)
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DB200_BUILT_FOR="{built_for}"', *(f"-I{p}" for p in includes), str(src), "-o", str(made), f"-L{base / 'lib'}", "-ltorch_python", "-ltorch",
           "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        made.unlink(missing_ok=True)
        raise RuntimeError(f"{cmd[0]} failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    os.replace(made, CALLS_PATH)
    return CALLS_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
    sys.exit(0 if CALLS_PATH.exists() else 1)
