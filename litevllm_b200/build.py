"""Build liblitekern.so (the sm_100a kernels + C ABI) in-tree with nvcc.

    python -m litevllm_b200.build          # incremental
    python -m litevllm_b200.build --force  # rebuild everything

Objects go to litevllm_b200/_build/, the shared library to
litevllm_b200/liblitekern.so, next to the ctypes loader that opens it, and the
CPython binding of csrc/spec_binding.cpp to litevllm_b200/_spec.so.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "liblitekern.so"
SPEC = PKG / "_spec.so"
INCLUDE = PKG.parent / "include"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH_FLAGS + [
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC,-O2",
    "--expt-relaxed-constexpr",
    f"-I{INCLUDE}",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found; liblitekern.so cannot be built")


def _deps(src: Path) -> list[Path]:
    return [src] + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted(INCLUDE.glob("*.h"))


def build(force: bool = False, verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    srcs = sorted(CSRC.glob("*.cu"))
    cc = nvcc()
    jobs = []
    for src in srcs:
        obj = BUILD / (src.stem + ".o")
        newest = max(p.stat().st_mtime for p in _deps(src))
        if force or not obj.exists() or obj.stat().st_mtime < newest:
            jobs.append((src, obj))

    def compile_one(job):
        src, obj = job
        cmd = [cc, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stdout}\n{res.stderr}")
        return obj

    with ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as ex:
        list(ex.map(compile_one, jobs))

    objs = [BUILD / (s.stem + ".o") for s in srcs]
    if force or jobs or not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [cc, *ARCH_FLAGS, "-shared", "-Xcompiler", "-fPIC", *map(str, objs), "-o", str(tmp)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc link failed:\n{res.stdout}\n{res.stderr}")
        os.replace(tmp, LIB)
    build_spec(force, verbose)
    return LIB


def build_spec(force: bool = False, verbose: bool = False) -> Path:
    """The binding, with g++ against the installed torch; liblitekern.so comes first.
    It is built again when its sources, torch, Python or the command change: the
    file beside the objects holds what the last one was built with."""
    import torch

    src = CSRC / "spec_binding.cpp"
    troot = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    tmp = SPEC.with_suffix(".so.tmp")
    cmd = [
        os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-fPIC", "-shared", f"-I{INCLUDE}",
        f'-DLK_TORCH_VERSION="{torch.__version__}"',
        f"-I{troot}/include", f"-I{troot}/include/torch/csrc/api/include", f"-I{cuda}/include",
        f"-I{sysconfig.get_paths()['include']}", str(src), "-o", str(tmp), f"-L{PKG}",
        "-l:liblitekern.so", f"-L{troot}/lib", "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10",
        "-Wl,-rpath,$ORIGIN",
    ]
    built_with = BUILD / "_spec.txt"
    key = "\n".join([sys.version, str(sysconfig.get_config_var("SOABI")), *cmd])
    newest = max(p.stat().st_mtime for p in [src, *INCLUDE.glob("*.h")])
    if (not force and SPEC.exists() and SPEC.stat().st_mtime >= newest and built_with.exists()
            and built_with.read_text() == key):
        return SPEC
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on {src.name}:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, SPEC)
    BUILD.mkdir(exist_ok=True)
    built_with.write_text(key)
    return SPEC


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args(argv)
    print(build(force=a.force, verbose=a.verbose))
    return 0


if __name__ == "__main__":
    sys.exit(main())
