"""Build recipe for libsrdit_b200.so (the C-ABI library of the sm_100a kernels).

Compiles every ``csrc/*.cu`` with nvcc for ``sm_100a`` only and links them into
``lib/libsrdit_b200.so`` inside the package, so the built library travels with
the source tree; and ``csrc/torch_calls.cpp``, the short way from torch tensors to some of
its entry points, with g++ into ``lib/_srdit_calls.so``. ``python build.py`` or ``build()``
from Python.
"""
from __future__ import annotations

import os
import pathlib
import shutil
import subprocess
import sys

PKG = pathlib.Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIBDIR = PKG / "lib"
LIB = LIBDIR / "libsrdit_b200.so"
CALLS = LIBDIR / "_srdit_calls.so"
INCLUDE = PKG.parent / "include"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
              "--expt-relaxed-constexpr", "-Xptxas", "-v"]


def nvcc_path() -> str:
    cand = [os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"]
    for c in cand:
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found: the sm_100a kernels cannot be built")


def sources():
    return sorted(CSRC.glob("*.cu"))


def up_to_date() -> bool:
    if not LIB.exists() or not CALLS.exists():
        return False
    t = min(LIB.stat().st_mtime, CALLS.stat().st_mtime)
    deps = list(CSRC.glob("*")) + list(INCLUDE.glob("*.h"))
    return all(p.stat().st_mtime <= t for p in deps)


def build_calls() -> str:
    """Compile the extension of ``csrc/torch_calls.cpp`` against the installed torch; its log."""
    import sysconfig

    import torch

    root = pathlib.Path(torch.__file__).parent
    cuda = pathlib.Path(nvcc_path()).resolve().parents[1]
    tmp = CALLS.with_suffix(".so.tmp")
    includes = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
                cuda / "include", sysconfig.get_paths()["include"]]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *(x for i in includes for x in ("-isystem", str(i))), str(CSRC / "torch_calls.cpp"),
           "-o", str(tmp), f"-L{root / 'lib'}", "-ltorch_python", "-lc10", "-lc10_cuda",
           f"-Wl,-rpath,{root / 'lib'}"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for torch_calls.cpp:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, CALLS)
    return f"$ {' '.join(cmd)}\n{r.stdout}{r.stderr}"


def build(force: bool = False, verbose: bool = False) -> pathlib.Path:
    """Compile the library if any source is newer than it. Returns its path."""
    if not force and up_to_date():
        return LIB
    LIBDIR.mkdir(exist_ok=True)
    nvcc = nvcc_path()
    objdir = LIBDIR / "obj"
    objdir.mkdir(exist_ok=True)
    objs = []
    logs = []
    for src in sources():
        obj = objdir / (src.stem + ".o")
        cmd = [nvcc, *ARCH_FLAGS, *NVCC_FLAGS, "-I", str(INCLUDE), "-I", str(CSRC),
               "-c", str(src), "-o", str(obj)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        logs.append(f"$ {' '.join(cmd)}\n{r.stdout}{r.stderr}")
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
        objs.append(str(obj))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc, *ARCH_FLAGS, "-shared", "-o", str(tmp), *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    logs.append(build_calls())
    os.replace(tmp, LIB)
    (LIBDIR / "build.log").write_text("\n".join(logs))
    if verbose:
        print("\n".join(logs))
    return LIB


if __name__ == "__main__":
    p = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(p)
