"""Build the three in-tree shared libraries of the package.

* ``libfdl_b200.so``  -- the C ABI of ``include/fdl_kvcache.h`` (all CUDA
  kernels), compiled by nvcc for sm_100a only.  Depends on the CUDA runtime
  alone; no torch types cross this boundary.
* ``libfdl_torch.so`` -- ``torch.library`` registration of the ``fdl`` ops on
  top of that ABI (host C++ only), linked against ``libfdl_b200.so`` with an
  ``$ORIGIN`` rpath.  Needs libtorch, not Python.
* ``libfdl_direct.so`` -- the Python module that calls some of these operators
  without the dispatcher, linked against ``libfdl_torch.so``.

They land next to this file so they travel with the source tree.  Run as
``python -m fast_v2_b200.build`` or call :func:`build`.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
LIB_ABI = PKG / "libfdl_b200.so"
LIB_TORCH = PKG / "libfdl_torch.so"
LIB_DIRECT = PKG / "libfdl_direct.so"

NVCC_ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc() -> str:
    home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = Path(home) / "bin" / "nvcc"
    return str(cand) if cand.exists() else (shutil.which("nvcc") or "nvcc")


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"build step failed ({r.returncode}): {cmd[0]} ... {cmd[-1]}")
    if verbose and (r.stdout or r.stderr):
        print(r.stdout + r.stderr, flush=True)


def build_abi(force: bool = False, verbose: bool = False, ptxas_verbose: bool = False) -> Path:
    deps = sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + [INCLUDE / "fdl_kvcache.h"]
    if not force and not _stale(LIB_ABI, deps):
        return LIB_ABI
    cmd = [_nvcc(), *NVCC_ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-shared",
           "--expt-relaxed-constexpr", str(CSRC / "fdl_b200.cu"), "-o", str(LIB_ABI) + ".tmp"]
    if ptxas_verbose:
        cmd.insert(1, "-Xptxas=-v")
    _run(cmd, verbose)
    os.replace(str(LIB_ABI) + ".tmp", LIB_ABI)
    return LIB_ABI


def _build_host(source: str, target: Path, libs: list[str], incs: list[str], verbose: bool) -> None:
    import torch
    from torch.utils import cpp_extension as ce

    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
           "-DTORCH_API_INCLUDE_EXTENSION_H", str(CSRC / source), "-o", str(target) + ".tmp"]
    cmd += [f"-I{d}" for d in ce.include_paths(device_type="cuda") + incs]
    cmd += [f"-L{d}" for d in ce.library_paths(device_type="cuda")]
    cmd += [f"-L{PKG}", *libs, "-Wl,-rpath,$ORIGIN"]
    _run(cmd, verbose)
    os.replace(str(target) + ".tmp", target)


def build_torch(force: bool = False, verbose: bool = False) -> Path:
    deps = [CSRC / "torch_ops.cpp", CSRC / "torch_ops.h", INCLUDE / "fdl_kvcache.h", LIB_ABI]
    if force or _stale(LIB_TORCH, deps):
        _build_host("torch_ops.cpp", LIB_TORCH, ["-lfdl_b200", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu",
                                                 "-ltorch_cuda", "-lcudart"], [], verbose)
    return LIB_TORCH


def build_direct(force: bool = False, verbose: bool = False) -> Path:
    deps = [CSRC / "torch_direct.cpp", CSRC / "torch_ops.h", LIB_TORCH]
    if force or _stale(LIB_DIRECT, deps):
        _build_host("torch_direct.cpp", LIB_DIRECT, ["-lfdl_torch", "-lfdl_b200", "-lc10", "-ltorch", "-ltorch_cpu",
                                                     "-ltorch_python"], [sysconfig.get_paths()["include"]], verbose)
    return LIB_DIRECT


def build(force: bool = False, verbose: bool = False) -> tuple[Path, Path, Path]:
    return build_abi(force, verbose), build_torch(force, verbose), build_direct(force, verbose)


if __name__ == "__main__":
    force = "--force" in sys.argv
    for lib in build(force=force, verbose="-v" in sys.argv):
        print(lib)
