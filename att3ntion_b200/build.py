"""Builds the in-tree native libraries with nvcc / gcc.

    python -m att3ntion_b200.build            # build what is out of date
    python -m att3ntion_b200.build --force    # rebuild everything

Produces ``att3ntion_b200/libatt3_b200.so`` (CUDA kernels + C ABI, sm_100a only) and
``att3ntion_b200/_serve_native.so`` (torch binding of the serving entry points, g++).
nvcc cross-compiles without a GPU, so this also runs on a CPU-only machine.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OBJ = PKG / "_obj"
LIB = PKG / "libatt3_b200.so"
BINDING = PKG / "_serve_native.so"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-v",
]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; the CUDA kernels cannot be built")
    return exe


def _newer(target: Path, deps) -> bool:
    if not target.exists():
        return False
    t = target.stat().st_mtime
    return all(Path(d).stat().st_mtime <= t for d in deps)


def _compile(src: Path, headers, force: bool) -> Path:
    obj = OBJ / (src.stem + ".o")
    if not force and _newer(obj, [src, *headers]):
        return obj
    cmd = [_nvcc(), *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    (OBJ / (src.stem + ".ptxas.log")).write_text(r.stdout + r.stderr)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    return obj


def _cuda_home() -> Path:
    return Path(_nvcc()).resolve().parent.parent


def _has_torch() -> bool:
    try:
        import torch  # noqa: F401
    except ImportError:
        return False
    return True


def _compile_binding(force: bool) -> Path:
    """The torch binding's object; linked against the library afterwards."""
    import sysconfig

    import torch
    src, obj = CSRC / "serve_torch.cpp", OBJ / "serve_torch.o"
    if not force and _newer(obj, [src, PKG.parent / "include" / "att3_b200.h", Path(torch.__file__)]):
        return obj
    inc = Path(torch.__file__).parent / "include"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_serve_native", "-DTORCH_API_INCLUDE_EXTENSION_H",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-isystem", str(inc), "-isystem",
           str(inc / "torch" / "csrc" / "api" / "include"), "-isystem", str(_cuda_home() / "include"), "-isystem",
           sysconfig.get_paths()["include"], "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    return obj


def _link_binding(obj: Path, force: bool) -> None:
    import torch
    if not force and _newer(BINDING, [obj]):
        return
    libs = Path(torch.__file__).parent / "lib"
    cmd = ["g++", "-shared", "-o", str(BINDING), str(obj), f"-L{PKG}", "-l:libatt3_b200.so", "-Wl,-rpath,$ORIGIN", f"-L{libs}",
           f"-Wl,-rpath,{libs}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")


def build(force: bool = False, verbose: bool = False) -> Path:
    OBJ.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    headers = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [PKG.parent / "include" / "att3_b200.h"]
    with_torch = _has_torch()
    with cf.ThreadPoolExecutor(max_workers=min(8, len(sources) + 1)) as ex:
        binding = ex.submit(_compile_binding, force) if with_torch else None
        objs = list(ex.map(lambda s: _compile(s, headers, force), sources))
    if force or not _newer(LIB, objs):
        cmd = [_nvcc(), "-shared", "-o", str(LIB), *map(str, objs), "-Xcompiler", "-fPIC"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    if with_torch:                               # the library does not wait for it, nor fall with it
        _link_binding(binding.result(), force)
    else:
        print(f"no torch in this Python: {BINDING.name} is not built, the C library is", file=sys.stderr)
    if verbose:
        for s in sources:
            log = OBJ / (s.stem + ".ptxas.log")
            if log.exists():
                print(f"--- {s.name}\n{log.read_text()}")
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
