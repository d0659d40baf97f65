"""Builds libsparsemoe_b200.so (the C-ABI library) in-tree with nvcc for sm_100a,
and _operators.so, the Python entry of the stand-alone operators, with g++
against torch's headers.

Usage: python sparsemoe_b200/build.py   (loaded by path: the package import needs the built library)
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libsparsemoe_b200.so"
BINDING_SRC = PKG / "binding" / "operators.cpp"
BINDING = PKG / "_operators.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
              "--expt-relaxed-constexpr", "-I", str(PKG.parent / "include")]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[Path]:
    return sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cpp")))


def _compile(src: Path, extra: list[str]) -> Path:
    obj = BUILD / (src.name + ".o")
    deps = [src] + list(CSRC.glob("*.h")) + list(CSRC.glob("*.cuh")) + list((PKG.parent / "include").glob("*.h"))
    if obj.exists() and obj.stat().st_mtime >= max(d.stat().st_mtime for d in deps):
        return obj
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, *extra, "-c", str(src), "-o", str(obj)]
    if src.suffix == ".cpp":
        cmd = [nvcc(), "-x", "c++", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-I",
               str(PKG.parent / "include"), "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    return obj


def binding_stamp() -> str:
    """What the binding's binary depends on besides its sources: the torch and the Python it was built against."""
    import importlib.metadata
    return f"torch {importlib.metadata.version('torch')}, python {sys.version_info[0]}.{sys.version_info[1]}"


def build_binding() -> Path | None:
    """The Python entry: no CUDA code, calls the C ABI through addresses it is given.  None where there is no torch."""
    import importlib.util
    if importlib.util.find_spec("torch") is None:
        return None
    deps = [BINDING_SRC, PKG.parent / "include" / "sparsemoe_b200.h"]
    stamp = BUILD / (BINDING.name + ".stamp")
    if BINDING.exists() and BINDING.stat().st_mtime >= max(d.stat().st_mtime for d in deps) and \
            stamp.exists() and stamp.read_text() == binding_stamp():
        return BINDING
    import sysconfig
    torch = Path(importlib.util.find_spec("torch").origin).parent
    cuda = Path(nvcc()).resolve().parents[1] / "include"
    inc = [torch / "include", torch / "include" / "torch" / "csrc" / "api" / "include",
           Path(sysconfig.get_paths()["include"]), cuda, PKG.parent / "include"]
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", *(a for i in inc for a in ("-isystem", str(i))),
           str(BINDING_SRC), "-o", str(tmp), "-L", str(torch / "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu",
           "-ltorch_cuda", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {BINDING_SRC.name}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, BINDING)
    stamp.write_text(binding_stamp())
    return BINDING


def build(verbose: bool = False, extra: list[str] | None = None) -> Path:
    BUILD.mkdir(exist_ok=True)
    extra = extra or []
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        binding = ex.submit(build_binding)
        objs = list(ex.map(lambda s: _compile(s, extra), sources()))
    newest = max(o.stat().st_mtime for o in objs)
    if not LIB.exists() or LIB.stat().st_mtime < newest:
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs), "-lpthread"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    entry = binding.result()   # (the library stands without it)
    if verbose:
        print(f"built {LIB}" + (f" and {entry.name}" if entry else "; no torch, so no Python entry of the operators"))
    return LIB


if __name__ == "__main__":
    build(verbose=True, extra=sys.argv[1:])
