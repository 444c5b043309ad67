"""Build the package's native library (CUDA kernels + C ABI) for sm_100a.

    python fast-compressai_b200/build_native.py [--force]

Produces fast_compressai/_lib/libfcai_b200.so in-tree with nvcc
(``-gencode arch=compute_100a,code=sm_100a``) and, where torch is installed, beside
it with the host compiler the module that takes the pointwise layers' calls from
tensors to that library: _layers_host-<torch's version>.<the interpreter's ABI>.so,
so that another torch gets a module of its own.  Callers of the C ABI need the
library alone.  No GPU is needed to build.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

ROOT = Path(__file__).resolve().parent
CSRC = ROOT / "csrc"
INCLUDE = ROOT.parent / "include"
LIB_DIR = ROOT / "fast_compressai" / "_lib"
LIB = LIB_DIR / "libfcai_b200.so"
HOST_SOURCE = "layers_host.cpp"

SOURCES = [
    "warp_div.cu",
    "conv_tc.cu",
    "linear_tc.cu",
    "rowwise.cu",
]
HEADERS = ["fcai_common.h", "tc_ptx.h", "layers_common.cuh"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O2", "--expt-relaxed-constexpr"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found; the CUDA toolkit is required to build fast_compressai")


def _inputs() -> list[Path]:
    files = [CSRC / s for s in SOURCES] + [CSRC / h for h in HEADERS]
    files += sorted(INCLUDE.glob("*.h"))
    return files


def up_to_date() -> bool:
    if not LIB.exists():
        return False
    t = LIB.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in _inputs())


def _host_module() -> tuple[Path | None, str]:
    """The module for the running interpreter and its torch, or None and what is missing to build it."""
    try:
        import torch
    except ImportError:
        return None, "torch is not installed"
    if torch.version.cuda is None:
        return None, "torch is installed without CUDA"
    for header in (Path(torch.__file__).resolve().parent / "include" / "ATen" / "ATen.h",
                   Path(sysconfig.get_paths()["include"]) / "Python.h"):
        if not header.exists():
            return None, f"{header} is missing"
    if shutil.which(os.environ.get("CXX", "g++")) is None:
        return None, "there is no host compiler"
    return LIB_DIR / f"_layers_host-{torch.__version__}.{sysconfig.get_config_var('SOABI')}.so", ""


def _host_up_to_date(host: Path) -> bool:
    if not host.exists():
        return False
    t = host.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in [CSRC / HOST_SOURCE, INCLUDE / "fcai_layers.h", INCLUDE / "fcai_warp_div.h"])


def _build_host(host: Path, verbose: bool) -> None:
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parents[1]
    tmp = host.with_suffix(f".so.{os.getpid()}.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for inc in (root / "include", root / "include" / "torch" / "csrc" / "api" / "include", cuda / "include",
                Path(sysconfig.get_paths()["include"])):
        cmd += ["-isystem", str(inc)]
    cmd += [str(CSRC / HOST_SOURCE), "-o", str(tmp), "-L", str(root / "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu",
            "-ltorch_cuda", "-lc10", "-lc10_cuda", "-L", str(LIB_DIR), "-lfcai_b200", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, host)


def build(force: bool = False, verbose: bool = False) -> Path:
    if force or not up_to_date():
        _build_lib(verbose)
    host, missing = _host_module()
    if host is None:
        if verbose:
            print(f"the pointwise layers' module is not built: {missing}", flush=True)
    elif force or not _host_up_to_date(host):
        _build_host(host, verbose)
    return LIB


def _build_lib(verbose: bool) -> None:
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    nvcc = _nvcc()
    objdir = ROOT / "_build"
    objdir.mkdir(exist_ok=True)
    objs, running = [], []
    for src in SOURCES:  # the sources compile side by side
        obj = objdir / (Path(src).stem + ".o")
        cmd = [nvcc, *ARCH, *FLAGS, "-I", str(INCLUDE), "-c", str(CSRC / src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        running.append((cmd, subprocess.Popen(cmd)))
        objs.append(str(obj))
    for cmd, proc in running:
        proc.wait()
    for cmd, proc in running:
        if proc.returncode:
            raise subprocess.CalledProcessError(proc.returncode, cmd)
    tmp = LIB.with_suffix(f".so.{os.getpid()}.tmp")
    cmd = [nvcc, *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *objs]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    args = ap.parse_args(argv)
    print(build(force=args.force, verbose=True))
    return 0


if __name__ == "__main__":
    sys.exit(main())
