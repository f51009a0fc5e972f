"""Build libmxfp8.so and libmxfp8_checked.so (sm_100a) in-tree with nvcc, and
_native.so, the binding of the 4-bit and cache operators, with the host compiler.

    python mxfp8-quantizer_b200/build.py [--force] [--ptxas-verbose]

The library links the CUDA runtime statically and exports only the C ABI
of include/mxfp8.h, mxfp4.h and mxfp8_cache.h.  The checked build compiles the same sources with
MXFP8_CHECKED (every global store tested against its output's bytes; see
include/mxfp8_checked.h).  nvcc cross-compiles, so this runs without a GPU.
The binding compiles against the installed torch and calls the library by the
addresses it is given, so it links neither to it nor to the CUDA runtime.
"""

from __future__ import annotations

import argparse
import os
import pathlib
import shutil
import subprocess
import sys
import sysconfig

PKG = pathlib.Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libmxfp8.so"
CHECKED_LIB = PKG / "libmxfp8_checked.so"
NATIVE = PKG / "_native.so"
BINDING = CSRC / "binding.cpp"
SOURCES = ["capi.cu", "quantize_tma.cu", "quantize_generic.cu", "dequantize.cu", "selftest.cu",
           "capi_mxfp4.cu", "mxfp4_convert.cu", "mxfp4_gemm.cu", "capi_cache.cu", "cache_copy.cu",
           "cache_attention.cu"]
HEADERS = ["ptx.cuh", "recipe.cuh", "launch.h", "guard.cuh", "tile.cuh", "row_path.cuh", "stores.cuh", "mxfp4.cuh",
           "tcgen05.cuh", "cache.cuh", "cache_index.h", "gemm_barriers.h"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and pathlib.Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the CUDA extension cannot be built")


def inputs() -> list[pathlib.Path]:
    return [CSRC / s for s in SOURCES] + [CSRC / h for h in HEADERS] + [
        ROOT / "include" / "mxfp8.h", ROOT / "include" / "mxfp8_checked.h", ROOT / "include" / "mxfp4.h",
        ROOT / "include" / "mxfp8_cache.h", pathlib.Path(__file__)]


def native_inputs() -> list[pathlib.Path]:
    return [BINDING, pathlib.Path(__file__)] + [ROOT / "include" / h for h in ("mxfp8.h", "mxfp4.h", "mxfp8_cache.h")]


def up_to_date(lib: pathlib.Path, sources: list[pathlib.Path]) -> bool:
    if not lib.exists():
        return False
    t = lib.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in sources)


def _command(out: pathlib.Path, checked: bool, verbose_ptxas: bool) -> list[str]:
    cmd = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-shared", "-Xcompiler", "-fPIC,-fvisibility=hidden",
           "-Xcompiler", "-Wall", "-I", str(ROOT / "include"), "-o", str(out)]
    if checked:
        cmd.append("-DMXFP8_CHECKED")
    if verbose_ptxas:
        cmd += ["-Xptxas", "-v"]
    return cmd + [str(CSRC / s) for s in SOURCES]


def _native_command(out: pathlib.Path) -> list[str]:
    """The host compiler on binding.cpp, with the flags torch's headers want."""
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    cuda_include = pathlib.Path(nvcc()).resolve().parent.parent / "include"
    # g++ as nvcc finds it: it must link the libstdc++ that torch runs on, as a shared library
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for path in [*include_paths(), sysconfig.get_paths()["include"], str(cuda_include)]:
        cmd += ["-isystem", path]
    cmd += ["-I", str(ROOT / "include"), "-o", str(out), str(BINDING)]
    for path in library_paths():
        cmd += ["-L", path]
    return cmd + ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"]


def build(force: bool = False, verbose_ptxas: bool = False) -> pathlib.Path:
    """Build what has a newer source (in parallel); returns the product library."""
    jobs = []

    def start(lib: pathlib.Path, sources: list[pathlib.Path], command) -> None:
        if force or not up_to_date(lib, sources):
            tmp = lib.with_name(f".{lib.stem}.{os.getpid()}.so")
            jobs.append((lib, tmp, subprocess.Popen(command(tmp), stdout=subprocess.PIPE, stderr=subprocess.PIPE,
                                                    text=True)))

    start(LIB, inputs(), lambda tmp: _command(tmp, False, verbose_ptxas))
    start(CHECKED_LIB, inputs(), lambda tmp: _command(tmp, True, False))
    start(NATIVE, native_inputs(), _native_command)
    failed = []
    for lib, tmp, proc in jobs:
        out, err = proc.communicate()
        if proc.returncode != 0:
            sys.stderr.write(out + err)
            failed.append(lib.name)
            continue
        if verbose_ptxas:
            sys.stderr.write(err)
        os.replace(tmp, lib)
    if failed:
        raise RuntimeError(f"the compiler failed building {', '.join(failed)}")
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--ptxas-verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose_ptxas=a.ptxas_verbose))
