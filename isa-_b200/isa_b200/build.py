"""Build the sm_100a C-ABI library ``libcimekv.so`` and its C++ tensor binding
``cimekv_torch.<torch version>.<python>.so`` in-tree.

    python -m isa_b200.build                  (or isa_b200.build.build_library())
    python -m isa_b200.build --library-only   the C ABI alone, which needs nvcc and nothing else

nvcc cross-compiles for sm_100a without a GPU.  Both land next to this file in
``_lib/`` so they travel with the source tree.  The binding's name says which torch
and Python it is for: another one finds none and builds its own.
"""

from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
SRC_DIR = PKG_DIR.parent / "csrc"
REPO_ROOT = PKG_DIR.parent.parent
INCLUDE_DIR = REPO_ROOT / "include"
LIB_DIR = PKG_DIR / "_lib"
LIB_PATH = LIB_DIR / "libcimekv.so"
DEBUG_LIB_PATH = LIB_DIR / "libcimekv_debug.so"  # table-index bounds checks (CIMEKV_DEBUG_BOUNDS=1)

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared", "--threads", "0",
]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libcimekv")
    return cand


def sources() -> list[Path]:
    return sorted(SRC_DIR.glob("*.cu"))


def binding_path() -> Path:
    """Where the tensor binding for this torch and this Python is."""
    import torch

    return LIB_DIR / f"cimekv_torch.{torch.__version__}.{sys.implementation.cache_tag}.so"


def build_library(force: bool = False, verbose: bool = False, debug: bool = False, binding: bool = True) -> Path:
    """Compile csrc/*.cu into _lib/libcimekv.so (or the bounds-checking
    libcimekv_debug.so with debug=True); skipped when up to date.  After the release
    library comes the tensor binding, unless ``binding`` is False or there is no torch or
    no C++ compiler to build it with (its operators then say that it is missing)."""
    out = _compile_library(force, verbose, debug)
    if binding and not debug:
        missing = [what for what, there in (("torch", importlib.util.find_spec("torch")), ("g++", shutil.which("g++")))
                   if not there]
        if missing:
            print(f"{' and '.join(missing)} not found: the library is built, its tensor binding is not", file=sys.stderr)
        else:
            build_binding(force)
    return out


def _compile_library(force: bool, verbose: bool, debug: bool) -> Path:
    srcs = sources()
    deps = srcs + sorted(INCLUDE_DIR.glob("*.h")) + sorted(SRC_DIR.glob("*.cuh"))
    out = DEBUG_LIB_PATH if debug else LIB_PATH
    if not force and out.exists():
        mtime = out.stat().st_mtime
        if all(p.stat().st_mtime <= mtime for p in deps):
            return out
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    tmp = out.with_suffix(".so.tmp")
    cmd = [_nvcc(), *NVCC_FLAGS, f"-I{INCLUDE_DIR}", f"-I{SRC_DIR}", *map(str, srcs), "-o", str(tmp)]
    if debug:
        cmd.insert(1, "-DCIMEKV_DEBUG_BOUNDS=1")
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, out)
    return out


def build_binding(force: bool = False) -> Path:
    """Compile csrc/torch_binding.cpp into binding_path(); skipped when up to date."""
    src, out = SRC_DIR / "torch_binding.cpp", binding_path()
    deps = [src, *INCLUDE_DIR.glob("*.h")]
    if not force and out.exists() and all(p.stat().st_mtime <= out.stat().st_mtime for p in deps):
        return out
    import torch
    from torch.utils.cpp_extension import include_paths

    cxx = shutil.which("g++")
    if cxx is None:
        raise RuntimeError("g++ not found: a C++ compiler is required to build the tensor binding")
    torch_lib = Path(torch.__file__).resolve().parent / "lib"
    cuda = Path(_nvcc()).resolve().parent.parent / "include"
    includes = [*include_paths("cuda"), sysconfig.get_paths()["include"], str(cuda)]
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    tmp = out.with_suffix(".so.tmp")
    subprocess.run([cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-DTORCH_EXTENSION_NAME=cimekv_torch",
                    f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                    *(f"-isystem{p}" for p in includes), f"-I{INCLUDE_DIR}", str(src), "-o", str(tmp), f"-L{torch_lib}",
                    "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"], check=True)
    os.replace(tmp, out)
    return out


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose="-v" in sys.argv, debug="--debug" in sys.argv,
                        binding="--library-only" not in sys.argv))
