"""Builds libnzb200.so in-tree (nvcc, sm_100a).

Run as ``python -m neuralzip_b200.build``. Besides the library, a small
extension module (nz_paged_torch.*.so, from csrc/nz_paged_torch.cpp against the
installed torch, and for that one alone) shortens Python's way to the paged-cache operators. The library holds the host packer
(C++) and the tile decode kernel (CUDA) behind the C ABI of
``include/nz_b200.h``; it is written next to this file under ``_lib/`` so a
snapshot of the repository carries it.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
ROOT = PACKAGE.parent
CSRC = PACKAGE / "csrc"
OUTPUT = PACKAGE / "_lib" / "libnzb200.so"
TORCH_CALLS_SOURCE = CSRC / "nz_paged_torch.cpp"
SOURCES = ("nz_host.cpp", "nz_huff0.cpp", "nz_storage.cpp", "nz_setup.cpp", "nz_schedule.cpp", "nz_decode.cu",
           "nz_pages.cu", "nz_rotary.cu", "nz_paged_attention.cu")
HEADERS = (ROOT / "include" / "nz_b200.h", CSRC / "nz_internal.h", CSRC / "nz_paged.h")
ARCH = ("-gencode", "arch=compute_100a,code=sm_100a")


def nvcc():
    for candidate in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if candidate and Path(candidate).exists():
            return candidate
    raise RuntimeError("nvcc was not found; set NVCC or put CUDA's bin directory on PATH.")


def _stale(output=None, inputs=None):
    output = OUTPUT if output is None else output
    if not output.exists():
        return True
    built = output.stat().st_mtime
    if inputs is None:
        inputs = [CSRC / name for name in SOURCES] + list(HEADERS) + [Path(__file__)]
    return any(path.stat().st_mtime > built for path in inputs)


def torch_calls():
    """Where the extension module of the torch calls lies, built or not: its
    name has the Python and the torch that it is for, since the code has the
    layout of their objects in it and would load, and misread them, under others."""
    import torch

    return OUTPUT.with_name(f"nz_paged_torch.{sysconfig.get_config_var('SOABI')}.torch-{torch.__version__}.so")


def build_torch_calls(force=False):
    """Compiles the torch calls (no CUDA code) when their source is newer; returns the module's path."""
    output = torch_calls()
    if not force and not _stale(output, [TORCH_CALLS_SOURCE, HEADERS[0], Path(__file__)]):
        return output
    import torch
    from torch.utils import cpp_extension

    cuda = Path(nvcc()).resolve().parent.parent / "include"
    includes = [*cpp_extension.include_paths(), str(cuda), sysconfig.get_paths()["include"]]
    tmp = output.with_suffix(".so.tmp")
    command = [
        os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{ROOT / 'include'}",
        *(word for path in includes for word in ("-isystem", path)), str(TORCH_CALLS_SOURCE),
        f"-L{Path(torch.__file__).parent / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-ltorch",
        "-o", str(tmp),
    ]
    result = subprocess.run(command, capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError(f"g++ failed ({result.returncode}):\n{result.stdout}\n{result.stderr}")
    os.replace(tmp, output)
    return output


def build(force=False, verbose=False, extra=()):
    """Compiles the library, then the torch calls, where a source is newer; returns the library's path.

    The torch calls only save time: without them (no g++, no headers of
    torch or Python) every call of the paged operators is checked."""
    OUTPUT.parent.mkdir(parents=True, exist_ok=True)
    if force or _stale():
        _build_library(verbose, extra)
    try:
        build_torch_calls(force)
    except (ImportError, OSError, RuntimeError) as error:
        for older in OUTPUT.parent.glob("nz_paged_torch.*"):  # than this library
            older.unlink()
        warnings.warn(f"{TORCH_CALLS_SOURCE.name} was not built, so calls of the paged operators take longer: {error}",
                      stacklevel=2)
    return OUTPUT


def _build_library(verbose, extra):
    tmp = OUTPUT.with_suffix(".so.tmp")
    command = [
        nvcc(), *ARCH, "-lineinfo", "-O3", "-std=c++17", "-shared", "--threads", "0",
        "-Xcompiler", "-fPIC,-O3,-pthread",
        "-Xptxas", "-v" if verbose else "-O3",
        f"-I{ROOT / 'include'}", f"-I{CSRC}",
        *extra,
        "-o", str(tmp),
        *(str(CSRC / name) for name in SOURCES),
    ]
    result = subprocess.run(command, capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError(f"nvcc failed ({result.returncode}):\n{result.stdout}\n{result.stderr}")
    if verbose:
        sys.stderr.write(result.stdout + result.stderr)
    os.replace(tmp, OUTPUT)


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(path)
