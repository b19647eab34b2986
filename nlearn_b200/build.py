"""Build the sm_100a kernel library ``libnl_ops.so`` in-tree with nvcc.

Each ``csrc/*.cu`` is compiled to an object under ``_build/`` (in parallel,
skipped when up to date) and linked into ``nlearn_b200/libnl_ops.so`` with the
static CUDA runtime, so the library depends only on the driver at run time.
``csrc/host/ops_py.cpp``, the host side of the serving operators, is compiled
with g++ against torch's headers into the extension module
``nlearn_b200/_ops.so``, which calls the library.

    python -m nlearn_b200.build          # or __graft_entry__.build()
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
INCLUDE = PKG.parent / "include"
OUT = PKG / "libnl_ops.so"
EXT_SRC = CSRC / "host" / "ops_py.cpp"
EXT = PKG / "_ops.so"
BUILD_DIR = PKG.parent / "_build"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
         "--expt-relaxed-constexpr", "-diag-suppress", "177"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: cannot build the sm_100a kernel library")


def _deps_mtime() -> float:
    files = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h"))
    return max((f.stat().st_mtime for f in files), default=0.0)


def _compile(nvcc: str, src: Path, obj: Path, dep_mtime: float, verbose: bool) -> str:
    if obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, dep_mtime):
        return f"up to date: {src.name}"
    cmd = [nvcc, *ARCH, *FLAGS, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
    return f"compiled: {src.name}" + (f"\n{r.stderr}" if verbose and r.stderr else "")


def _ext_made_for() -> str:
    """What the extension module is compiled against besides its sources: torch's headers and Python's."""
    import torch
    return f"torch {torch.__version__} {Path(torch.__file__).resolve().parent} python {sys.version}"


def _build_ext() -> str:
    """The extension module (linked against libnl_ops.so, which lies beside it)."""
    import torch
    newest = max(EXT_SRC.stat().st_mtime, (INCLUDE / "nl_ops.h").stat().st_mtime)
    stamp, made_for = BUILD_DIR / "ops_py.made_for", _ext_made_for()
    if (EXT.exists() and EXT.stat().st_mtime >= newest and stamp.exists() and stamp.read_text() == made_for):
        return f"up to date: {EXT_SRC.name}"
    tdir = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parents[1] / "include"
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-w",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f"-I{sysconfig.get_paths()['include']}",
           f"-I{tdir / 'include'}", f"-I{tdir / 'include' / 'torch' / 'csrc' / 'api' / 'include'}", f"-I{cuda}",
           str(EXT_SRC), "-o", str(EXT), f"-L{PKG}", "-lnl_ops", f"-L{tdir / 'lib'}", "-ltorch_python", "-ltorch_cpu",
           "-ltorch", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {EXT_SRC.name}:\n{r.stdout}\n{r.stderr}")
    stamp.write_text(made_for)
    return f"compiled: {EXT_SRC.name}"


def build(verbose: bool = False) -> Path:
    nvcc = _nvcc()
    BUILD_DIR.mkdir(exist_ok=True)
    srcs = sorted(CSRC.glob("*.cu"))
    dep = _deps_mtime()
    objs = [BUILD_DIR / (s.stem + ".o") for s in srcs]
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        for msg in ex.map(lambda so: _compile(nvcc, so[0], so[1], dep, verbose), zip(srcs, objs)):
            if verbose:
                print(msg)
    newest = max(o.stat().st_mtime for o in objs)
    if not OUT.exists() or OUT.stat().st_mtime < newest:
        cmd = [nvcc, *ARCH, "-shared", "-cudart", "static", "-o", str(OUT), *map(str, objs)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    msg = _build_ext()
    if verbose:
        print(msg)
    return OUT


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
