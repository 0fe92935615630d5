"""Build libla_attention.so (sm_100a) in-tree with nvcc, and its torch binding.

    python -m trainium_linear_attention_b200.build [--force] [--verbose]

Every ``csrc/*.cu`` is compiled with
``-gencode arch=compute_100a,code=sm_100a -lineinfo -O3`` into ``_build/`` and
linked into ``trainium_linear_attention_b200/lib/libla_attention.so``.  The
CUDA runtime is linked statically; the CUDA driver is reached at run time
through ``cudaGetDriverEntryPoint`` (TMA descriptors), so the library has no
link-time dependency on ``libcuda``.  ``csrc/torch_binding.cpp`` becomes
``lib/_la_torch.*.so``, named for the interpreter and the torch that it is built
for (g++, torch's headers; it has no kernels and takes the C entry points from
the library at run time).  Objects are rebuilt only when a source or header is
newer than they are.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
BUILD = ROOT / "_build"
LIB = PKG / "lib" / "libla_attention.so"
BINDING_SRC = CSRC / "torch_binding.cpp"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
CFLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O3",
          "--expt-relaxed-constexpr", "-I" + str(INCLUDE), "-I" + str(CSRC)]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found (set $NVCC)")


def _headers_mtime() -> float:
    hs = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h"))
    return max((h.stat().st_mtime for h in hs), default=0.0)


def _compile(src: Path, obj: Path, verbose: bool) -> str:
    cmd = [nvcc(), *ARCH_FLAGS, *CFLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    return res.stderr if verbose else ""


def _build_binding(force: bool) -> None:
    """Compile the torch binding (no CUDA code: the C++ compiler alone)."""
    import torch

    from . import _torch_binding
    binding = _torch_binding.path()
    newest = max(f.stat().st_mtime for f in (BINDING_SRC, INCLUDE / "la_attention.h",
                                             Path(__file__)))  # (which has the command)
    if not force and binding.exists() and binding.stat().st_mtime >= newest:
        return
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parents[1]
    tmp = binding.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-I" + str(INCLUDE),
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for path in (root / "include", root / "include/torch/csrc/api/include", cuda / "include",
                 sysconfig.get_path("include")):
        cmd += ["-isystem", str(path)]
    cmd += [str(BINDING_SRC), "-o", str(tmp), f"-L{root / 'lib'}", f"-Wl,-rpath,{root / 'lib'}",
            "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed for {BINDING_SRC.name}:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, binding)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every kernel source, link the shared library and compile the torch
    binding; returns the library's path.  A binding that cannot be built is an error
    behind the linking: the library is there for C all the same."""
    BUILD.mkdir(exist_ok=True)
    LIB.parent.mkdir(exist_ok=True)
    hdr = _headers_mtime()
    srcs = sorted(CSRC.glob("*.cu"))
    jobs = []
    for src in srcs:
        obj = BUILD / (src.stem + ".o")
        if force or not obj.exists() or obj.stat().st_mtime < max(src.stat().st_mtime, hdr):
            jobs.append((src, obj))
    with cf.ThreadPoolExecutor(max_workers=min(8, len(jobs) + 1)) as ex:
        binding = ex.submit(_build_binding, force)
        for out in ex.map(lambda j: _compile(j[0], j[1], verbose), jobs):
            if out:
                print(out, file=sys.stderr)
        objs = [BUILD / (s.stem + ".o") for s in srcs]
        newest = max(o.stat().st_mtime for o in objs)
        if force or jobs or not LIB.exists() or LIB.stat().st_mtime < newest:
            tmp = LIB.with_suffix(".so.tmp")
            cmd = [nvcc(), *ARCH_FLAGS, "-shared", "-o", str(tmp), *map(str, objs)]
            res = subprocess.run(cmd, capture_output=True, text=True)
            if res.returncode != 0:
                raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
            os.replace(tmp, LIB)
        binding.result()
    return LIB


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true", help="print ptxas register/smem usage")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))


if __name__ == "__main__":
    main()
