"""Build libltx_hip.so (gfx950) in-tree from csrc/*.hip.

Usage: python ltx-2-mlx_amd/build_lib.py [--jobs N]

Each translation unit is compiled to an object with hipcc, then linked into
ltx-2-mlx_amd/ltx_amd/libltx_hip.so, which the ctypes loader in
ltx_amd/_lib.py opens; csrc/calls.cpp, the native host side of small calls,
becomes ltx_amd/_calls.so.  The build always recompiles (it is the "does it
build" check) and writes to a temporary name first, so a failed build never
leaves a half-written library behind.
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

PKG_ROOT = Path(__file__).resolve().parent
CSRC = PKG_ROOT / "csrc"
OBJ_DIR = PKG_ROOT / "_build"
LIB_PATH = PKG_ROOT / "ltx_amd" / "libltx_hip.so"
ARCH = "gfx950"

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # Packed-fp32 VALU forms stay disabled for every kernel in this library.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.hip"))


def _compile(src: Path) -> Path:
    obj = OBJ_DIR / (src.stem + ".o")
    cmd = [hipcc(), *HIPCC_FLAGS, "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{proc.stderr}")
    return obj


def build_calls() -> Path | None:
    """ltx_amd/_calls.so: the native host calls (a CPython module on torch's
    headers; the kernels stay behind the C ABI).  Without a host compiler or the
    headers of Python and torch there is none (an earlier one goes too): the same
    calls then run through Python."""
    import torch
    from torch.utils.cpp_extension import include_paths

    lib_dir = Path(torch.__file__).parent / "lib"
    out = LIB_PATH.with_name("_calls.so")
    tmp = out.with_suffix(".so.tmp")
    python_include = Path(sysconfig.get_paths()["include"])
    compiler = next((c for c in ("g++", "clang++", "/opt/rocm/llvm/bin/clang++") if shutil.which(c)), None)
    torch_header = "torch/csrc/autograd/python_variable.h"
    missing = ("a C++ compiler" if compiler is None else
               f"{python_include}/Python.h" if not (python_include / "Python.h").exists() else
               torch_header if not any((Path(p) / torch_header).exists() for p in include_paths()) else None)
    if missing:
        out.unlink(missing_ok=True)
        print(f"no {missing}: {out.name} is not built, small MXFP4, int8, rotary and per-head norm calls go through Python")
        return None
    cmd = [compiler, "-O2", "-std=c++17", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DLTX_CALLS_BUILT_FOR="torch {torch.__version__}, Python {sys.version_info[0]}.{sys.version_info[1]}"',
           *(f for p in include_paths() for f in ("-isystem", p)), f"-I{python_include}",
           str(CSRC / "calls.cpp"), "-o", str(tmp), f"-L{lib_dir}", "-ltorch_python", "-ltorch_cpu", "-lc10",
           f"-Wl,-rpath,{lib_dir}"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{compiler} failed for calls.cpp:\n{proc.stderr}")
    os.replace(tmp, out)
    return out


def build(jobs: int | None = None, verbose: bool = True) -> Path:
    OBJ_DIR.mkdir(exist_ok=True)
    srcs = sources()
    if not srcs:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    jobs = jobs or min(len(srcs) + 1, os.cpu_count() or 4, 8)
    with cf.ThreadPoolExecutor(max_workers=jobs) as pool:
        calls = pool.submit(build_calls)
        objs = list(pool.map(_compile, srcs))
        calls.result()
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stderr}")
    os.replace(tmp, LIB_PATH)
    if verbose:
        print(f"built {LIB_PATH} from {len(srcs)} sources", flush=True)
    return LIB_PATH


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--jobs", type=int, default=None)
    args = ap.parse_args(argv)
    build(args.jobs)
    return 0


if __name__ == "__main__":
    sys.exit(main())
