"""Build librustane_cuda.so (sm_100a) in-tree.

Every `.cu` / `.cpp` file under ``rustane_b200/csrc`` is compiled by nvcc for
``-gencode arch=compute_100a,code=sm_100a`` and linked into
``rustane_b200/librustane_cuda.so`` with the static CUDA runtime.  Objects are
cached under ``rustane_b200/_build`` and rebuilt when a source or header is
newer.  ``rustane_b200/csrc_torch/ops.cpp`` (the torch binding of the serving
operators) is compiled by the host compiler against the installed torch, where there is one, into
``rustane_b200/_torch_ops<suffix>.so``.  No GPU is needed to build.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "librustane_cuda.so"
INCLUDE = PKG.parent / "include"
TORCH_SRC = PKG / "csrc_torch" / "ops.cpp"
TORCH_EXT = PKG / f"_torch_ops{sysconfig.get_config_var('EXT_SUFFIX')}"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
              "--expt-relaxed-constexpr", "-I", str(CSRC), "-I", str(INCLUDE)]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build librustane_cuda.so")
    return cand


def _headers() -> list[Path]:
    return sorted(list(CSRC.glob("*.h")) + list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h")))


def _compile(src: Path, verbose: bool) -> Path:
    obj = BUILD / (src.name + ".o")
    newest_dep = max([src.stat().st_mtime] + [h.stat().st_mtime for h in _headers()])
    if obj.exists() and obj.stat().st_mtime >= newest_dep:
        return obj
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
    if src.suffix == ".cpp":
        cmd = [nvcc(), *NVCC_FLAGS, "-x", "cu", *ARCH, "-c", str(src), "-o", str(obj)]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    return obj


def build_torch_ext(verbose: bool = False) -> Path | None:
    """The torch binding; links librustane_cuda.so (found next to it at run time).  None without torch: the
    C library does not need it.  Built again when its sources, torch or the command are others than before."""
    try:
        import torch
    except ImportError:
        print(f"torch is not installed: {TORCH_EXT.name} (rustane_b200.ops) is not built")
        return None
    root = Path(torch.__file__).parent
    cuda = Path(nvcc()).resolve().parent.parent / "include"
    inc = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", cuda, INCLUDE,
           sysconfig.get_paths()["include"]]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-w",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-DTORCH_EXTENSION_NAME=_torch_ops",
           *(f"-isystem{i}" for i in inc), str(TORCH_SRC), "-o", str(TORCH_EXT), f"-L{PKG}", "-l:librustane_cuda.so",
           f"-L{root / 'lib'}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
    newest = max([TORCH_SRC.stat().st_mtime] + [h.stat().st_mtime for h in INCLUDE.glob("*.h")])
    made_by, how = BUILD / "torch_ops.txt", f"torch {torch.__version__}\n{' '.join(cmd)}\n"
    if TORCH_EXT.exists() and TORCH_EXT.stat().st_mtime >= newest and made_by.exists() and made_by.read_text() == how:
        return TORCH_EXT
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for {TORCH_SRC.name}:\n{res.stdout}\n{res.stderr}")
    made_by.write_text(how)
    return TORCH_EXT


def build(verbose: bool = False, jobs: int | None = None) -> Path:
    BUILD.mkdir(exist_ok=True)
    sources = sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cpp")))
    jobs = jobs or min(len(sources), os.cpu_count() or 4)
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), sources))
    newest = max(o.stat().st_mtime for o in objs)
    if not LIB.exists() or LIB.stat().st_mtime < newest:
        cmd = [nvcc(), *ARCH, "-shared", "-o", str(LIB), *map(str, objs), "-ldl", "-lpthread", "-lrt"]
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    build_torch_ext(verbose)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
