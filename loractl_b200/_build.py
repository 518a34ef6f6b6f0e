"""Builds libloractl_b200.so in-tree with nvcc for sm_100a.

Usage: `python -m loractl_b200._build` (or `__graft_entry__.build()`).  nvcc
cross-compiles without a GPU; the resulting `lib/libloractl_b200.so` is what
`loractl_b200._lib` loads.  Every translation unit is compiled to its own object
(in parallel, and only when it or a header changed), then linked; internal C++
symbols are hidden, only the C ABI of include/loractl_b200.h is exported.  The PyTorch binding of the
short calls (`lib/_lq_torch.*.so`, csrc/lq_torch.cpp) is built with g++ against the installed torch.
"""
from __future__ import annotations

import concurrent.futures
import importlib.metadata
import pathlib
import shutil
import subprocess
import sys

PKG = pathlib.Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OBJ = PKG / "lib" / "obj"
LIB = PKG / "lib" / "libloractl_b200.so"
HEADER = PKG.parent / "include" / "loractl_b200.h"
SOURCES = ["lq_api.cu", "lq_quant.cu", "lq_simt.cu", "lq_tc.cu", "lq_w4.cu", "lq_prof.cu", "lq_step.cu", "lq_fused.cu", "lq_bwd_small.cu",
           "lq_block.cu", "lq_resnorm.cu", "lq_gradnorm.cu", "lq_mx4.cu"]
# the PyTorch binding of the short calls: a Python module that links the library and torch
TORCH_SRC = CSRC / "lq_torch.cpp"
FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
]


def _headers_mtime() -> float:
    return max(p.stat().st_mtime for p in [*CSRC.glob("*.cuh"), HEADER])


def _stale(out: pathlib.Path, deps_mtime: float) -> bool:
    return not out.exists() or out.stat().st_mtime < deps_mtime


def torch_module() -> pathlib.Path:
    """The binding for this Python and the installed torch, whose C++ internals it is compiled against: they stand in its name,
    so that another torch asks for a build of its own.  (torch itself is not imported.)"""
    return PKG / "lib" / f"_lq_torch.{sys.implementation.cache_tag}-torch{importlib.metadata.version('torch')}.so"


def _torch_module_stale() -> bool:
    return _stale(torch_module(), max(HEADER.stat().st_mtime, TORCH_SRC.stat().st_mtime))


def needs_build() -> bool:
    hdr = _headers_mtime()
    if _stale(LIB, hdr) or _torch_module_stale():
        return True
    return any((CSRC / s).stat().st_mtime > LIB.stat().st_mtime for s in SOURCES)


def _build_torch_module(force: bool) -> None:
    """g++ on csrc/lq_torch.cpp against the installed torch; finds the library beside itself."""
    if not force and not _torch_module_stale():
        return
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths

    libs = pathlib.Path(torch.__file__).resolve().parent / "lib"
    cuda = pathlib.Path(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc").resolve().parent.parent
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_lq_torch",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-I{p}" for p in [*include_paths(), sysconfig.get_paths()["include"], cuda / "include"]],
           "-o", str(torch_module()), str(TORCH_SRC), f"-L{LIB.parent}", f"-l:{LIB.name}", f"-L{libs}", "-lc10", "-lc10_cuda",
           "-ltorch", "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed on {TORCH_SRC.name} ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")


def build(force: bool = False, verbose: bool = False) -> pathlib.Path:
    if not force and not needs_build():
        return LIB
    stale_lib = force or _stale(LIB, _headers_mtime()) or any((CSRC / s).stat().st_mtime > LIB.stat().st_mtime for s in SOURCES)
    if not stale_lib:
        _build_torch_module(force)
        return LIB
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    OBJ.mkdir(parents=True, exist_ok=True)
    hdr = _headers_mtime()

    def compile_one(src: str):
        obj = OBJ / (src[:-3] + ".o")
        if not force and not _stale(obj, max(hdr, (CSRC / src).stat().st_mtime)):
            return obj, ""
        cmd = [nvcc, *FLAGS, *(["-Xptxas", "-v"] if verbose else []), "-c", "-o", str(obj), str(CSRC / src)]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src} ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
        return obj, proc.stderr

    with concurrent.futures.ThreadPoolExecutor(max_workers=len(SOURCES)) as pool:
        results = list(pool.map(compile_one, SOURCES))
    if verbose:
        for _, log in results:
            if log:
                print(log)
    link = [nvcc, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-Xlinker",
            f"--version-script={CSRC / 'exports.map'}", "-o", str(LIB), *[str(o) for o, _ in results]]
    proc = subprocess.run(link, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    _build_torch_module(force)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
