"""Build the liteweight_b200 CUDA library in-tree (sm_100a only).

    python -m liteweight_b200.build          # compiles csrc/*.cu -> _lib/liblw_b200.so
                                             # and csrc/bind_paged.cpp -> _lib/lw_bind.so

The library is a plain C-ABI shared object (include/liteweight_b200.h) with
the CUDA runtime linked statically, loaded from Python with ctypes. nvcc
cross-compiles for sm_100a without a GPU. lw_bind.so is a Python extension module
over that ABI for the calls whose argument handling in Python would cost more
than their launches; it is built by g++ against torch's headers.
"""

from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
LIB_DIR = PKG / "_lib"
LIB = LIB_DIR / "liblw_b200.so"
BIND_SRC = CSRC / "bind_paged.cpp"
BIND = LIB_DIR / "lw_bind.so"
STAMP = LIB_DIR / "liblw_b200.sha"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O3", "--expt-relaxed-constexpr",
         "-Xptxas", "-O3", "-cudart", "static"]
BIND_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-shared"]


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _digest() -> str:
    h = hashlib.sha256()
    for f in sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h")) + [BIND_SRC]):
        h.update(f.name.encode())
        h.update(f.read_bytes())
    # the extension module is tied to this interpreter and torch
    import torch
    h.update(" ".join(ARCH + FLAGS + BIND_FLAGS + [sys.version, torch.__version__]).encode())
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


def up_to_date() -> bool:
    return LIB.exists() and BIND.exists() and STAMP.exists() and STAMP.read_text().strip() == _digest()


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every csrc/*.cu for sm_100a, link liblw_b200.so and build lw_bind.so
    (skipped when up to date)."""
    if not force and up_to_date():
        return LIB
    LIB_DIR.mkdir(exist_ok=True)
    obj_dir = LIB_DIR / "obj"
    obj_dir.mkdir(exist_ok=True)
    cc = nvcc()
    objs, procs = [], []
    for src in sources():
        obj = obj_dir / (src.stem + ".o")
        cmd = [cc, *ARCH, *FLAGS, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        objs.append(obj)
    bind_tmp = BIND.with_suffix(".so.tmp")
    cmd = _bind_command(bind_tmp)
    if verbose:
        print(" ".join(cmd), flush=True)
    procs.append((BIND_SRC, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            failed.append(f"{src.name}:\n{out.decode(errors='replace')}")
        elif verbose and out:
            print(out.decode(errors="replace"))
    if failed:
        raise RuntimeError("the build failed\n" + "\n".join(failed))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [cc, *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objs), "-lrt", "-ldl", "-lpthread"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    os.replace(bind_tmp, BIND)
    STAMP.write_text(_digest())
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
