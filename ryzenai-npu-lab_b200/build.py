"""Build libb2attn.so in-tree with nvcc for sm_100a, and the native binding
_b2torch.so of its smallest calls with g++.

The shared library is the product's compute path: it holds every CUDA kernel
and the C ABI declared in the headers of include/.  It is built next to this file so that it travels with the source tree to the GPU host.
"""
from __future__ import annotations

import os
import pathlib
import shutil
import subprocess
import warnings

PKG = pathlib.Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libb2attn.so"
BINDING = PKG / "_b2torch.so"
BINDING_SOURCE = CSRC / "b2_torch.cpp"
BINDING_HEADERS = [ROOT / "include" / "b2_kv8.h", ROOT / "include" / "b2_tables.h"]
SOURCES = [CSRC / "b2_attn.cu", CSRC / "b2_block.cu", CSRC / "b2_gemm.cu",
           CSRC / "b2_kv8.cu", CSRC / "b2_tables.cu"]
HEADERS = [ROOT / "include" / "b2_decode_attn.h", ROOT / "include" / "b2_block.h",
           ROOT / "include" / "b2_kv8.h", ROOT / "include" / "b2_tables.h", CSRC / "b2_internal.h",
           CSRC / "b2_device.cuh"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC",
    "-Xptxas", "-v",
]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found")
    return path


def needs_build(lib: pathlib.Path = LIB) -> bool:
    if not lib.exists():
        return True
    mtime = lib.stat().st_mtime
    return any(p.stat().st_mtime > mtime for p in SOURCES + HEADERS)


def binding_stamp() -> str:
    """What the binding is compiled against and of no use without: this torch, this Python."""
    import sysconfig

    import torch
    return f"b2torch for torch {torch.__version__} and {sysconfig.get_config_var('SOABI')}"


def binding_matches(path: pathlib.Path = BINDING) -> bool:
    """Whether the binding at `path` was compiled against the installed torch and this Python (it carries their
    names, which are looked for before it is loaded)."""
    return path.exists() and binding_stamp().encode() in path.read_bytes()


def binding_needs_build() -> bool:
    if not binding_matches(BINDING):
        return True
    mtime = BINDING.stat().st_mtime
    return any(p.stat().st_mtime > mtime for p in (BINDING_SOURCE, *BINDING_HEADERS))


def _start_binding(force: bool):
    """The compilation of the binding against the installed torch, started; None when up to date."""
    if not force and not binding_needs_build():
        return None
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths
    tmp = BINDING.with_suffix(".so.tmp")
    lib = pathlib.Path(torch.__file__).parent / "lib"
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-DNDEBUG",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DB2_TORCH_STAMP="{binding_stamp()}"', f"-I{ROOT / 'include'}",
           *(f"-I{d}" for d in include_paths()), f"-I{sysconfig.get_paths()['include']}", str(BINDING_SOURCE),
           f"-L{lib}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-o", str(tmp)]
    return tmp, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)


def _finish_binding(started) -> None:
    if started is None:
        return
    tmp, proc = started
    text, _ = proc.communicate()
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed ({proc.returncode}):\n{text}")
    os.replace(tmp, BINDING)


def _without_binding(error: Exception) -> None:
    """The package works without the binding, which halves the host's time of its smallest calls: its failure is a
    warning, and a binding of other sources or another torch does not stay."""
    try:
        stale = binding_needs_build()
    except ImportError:
        stale = True
    if stale:
        BINDING.unlink(missing_ok=True)
    warnings.warn(f"{BINDING.name} was not built, its calls go through Python: {error}", stacklevel=3)


def build(force: bool = False, verbose: bool = False) -> pathlib.Path:
    """Compile the CUDA sources into libb2attn.so and the binding (each skipped when up to date)."""
    binding = None
    try:
        binding = _start_binding(force)
    except Exception as e:      # no torch, no compiler
        _without_binding(e)
    try:
        return _build_library(force, verbose)
    finally:
        try:
            _finish_binding(binding)
        except Exception as e:
            _without_binding(e)


def _build_library(force: bool, verbose: bool) -> pathlib.Path:
    if not force and not needs_build():
        return LIB
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc(), *NVCC_FLAGS, "-I", str(ROOT / "include"),
           *map(str, SOURCES), "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed ({proc.returncode}):\n{proc.stderr}")
    if verbose:
        print(proc.stderr)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    build(force=True, verbose=True)
    print(LIB)
