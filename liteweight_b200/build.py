"""Build the liteweight_b200 CUDA library in-tree (sm_100a only).

    python -m liteweight_b200.build          # compiles csrc/*.cu -> _lib/liblw_b200.so
                                             # and csrc/bind_paged.cpp -> _lib/lw_bind.so

The library is a plain C-ABI shared object (include/liteweight_b200.h) with
the CUDA runtime linked statically, loaded from Python with ctypes. nvcc
cross-compiles for sm_100a without a GPU. lw_bind.so is a Python extension module
over that ABI for the calls whose argument handling in Python would cost more
than their launches; it is built by g++ against torch's headers. The C library
alone needs neither torch nor Python's headers: `python liteweight_b200/build.py`
links it before it reports that the extension module could not be built.
"""

from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
LIB_DIR = PKG / "_lib"
LIB = LIB_DIR / "liblw_b200.so"
BIND_SRC = CSRC / "bind_paged.cpp"
BIND = LIB_DIR / "lw_bind.so"
STAMP = LIB_DIR / "liblw_b200.sha"
BIND_STAMP = LIB_DIR / "lw_bind.sha"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O3", "--expt-relaxed-constexpr",
         "-Xptxas", "-O3", "-cudart", "static"]
BIND_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-shared"]


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _digest() -> str:
    h = hashlib.sha256()
    for f in sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))):
        h.update(f.name.encode())
        h.update(f.read_bytes())
    h.update(" ".join(ARCH + FLAGS).encode())
    return h.hexdigest()


def _bind_digest() -> str:
    """The extension module is tied to this interpreter and torch."""
    import torch
    h = hashlib.sha256()
    for f in [BIND_SRC, *sorted(INCLUDE.glob("*.h"))]:
        h.update(f.read_bytes())
    h.update(" ".join(BIND_FLAGS + [sys.version, torch.__version__]).encode())
    return h.hexdigest()


def _bind_command(out: Path) -> list[str]:
    """g++ for the Python extension module against this interpreter and torch."""
    import torch
    root = Path(torch.__file__).resolve().parent
    includes = [INCLUDE, root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
                sysconfig.get_paths()["include"], Path(nvcc()).resolve().parent.parent / "include"]
    return ["g++", *BIND_FLAGS, f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *(f"-I{i}" for i in includes), str(BIND_SRC), "-o", str(out), f"-L{root / 'lib'}", "-ltorch_python", "-ltorch",
            "-ltorch_cpu", "-lc10", "-lc10_cuda"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the liteweight_b200 CUDA library cannot be built")


def _current(out: Path, stamp: Path, digest) -> bool:
    return out.exists() and stamp.exists() and stamp.read_text().strip() == digest()


def _library_current() -> bool:
    return _current(LIB, STAMP, _digest)


def _bind_current() -> bool:
    try:
        return _current(BIND, BIND_STAMP, _bind_digest)
    except ImportError:
        return False


def up_to_date() -> bool:
    return _library_current() and _bind_current()


def _build_library(cc: str, verbose: bool) -> None:
    obj_dir = LIB_DIR / "obj"
    obj_dir.mkdir(exist_ok=True)
    objs, procs = [], []
    for src in sources():
        obj = obj_dir / (src.stem + ".o")
        cmd = [cc, *ARCH, *FLAGS, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        objs.append(obj)
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            failed.append(f"{src.name}:\n{out.decode(errors='replace')}")
        elif verbose and out:
            print(out.decode(errors="replace"))
    if failed:
        raise RuntimeError("nvcc failed\n" + "\n".join(failed))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [cc, *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objs), "-lrt", "-ldl", "-lpthread"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    STAMP.write_text(_digest())


def _build_bind(verbose: bool) -> None:
    tmp = BIND.with_suffix(".so.tmp")
    try:
        cmd = _bind_command(tmp)
        if verbose:
            print(" ".join(cmd), flush=True)
        made = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
        why = made.stdout.decode(errors="replace") if made.returncode else None
    except (ImportError, AttributeError, OSError) as e:   # no torch, none that it can be built with, no compiler
        why = f"{type(e).__name__}: {e}"
    if why is not None:
        raise RuntimeError(f"{BIND_SRC.name}, the Python extension module, could not be built:\n{why}")
    os.replace(tmp, BIND)
    BIND_STAMP.write_text(_bind_digest())


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every csrc/*.cu for sm_100a, link liblw_b200.so and build lw_bind.so
    (each skipped when up to date). The C library needs neither torch nor Python:
    it is there when only the extension module fails."""
    if not force and up_to_date():
        return LIB
    LIB_DIR.mkdir(exist_ok=True)
    # side by side; the C library's failure is the one that is raised
    with ThreadPoolExecutor(1) as pool:
        bind = None if not force and _bind_current() else pool.submit(_build_bind, verbose)
        if force or not _library_current():
            _build_library(nvcc(), verbose)
        if bind is not None:
            bind.result()
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
