"""Build recipe for libsrdit_b200.so (the C-ABI library of the sm_100a kernels).

Compiles every ``csrc/*.cu`` with nvcc for ``sm_100a`` only and links them into
``lib/libsrdit_b200.so`` inside the package, so the built library travels with
the source tree; and, where that works, ``csrc/torch_calls.cpp``, the short way from torch
tensors to some of its entry points, with g++ into ``lib/_srdit_calls.<python>-<torch>.so``.
``python build.py`` or ``build()`` from Python.
"""
from __future__ import annotations

import os
import pathlib
import shutil
import subprocess
import sys
import warnings

PKG = pathlib.Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIBDIR = PKG / "lib"
LIB = LIBDIR / "libsrdit_b200.so"
CALLS_SRC = CSRC / "torch_calls.cpp"
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


def calls_path() -> pathlib.Path:
    """Where the extension for the running Python and torch is: it is built against both, so one
    for others is never loaded."""
    import torch

    return LIBDIR / f"_srdit_calls.{sys.implementation.cache_tag}-torch{torch.__version__}.so"


def newer(path: pathlib.Path, sources) -> bool:
    """Whether a file is there and no source was changed since."""
    return path.exists() and all(p.stat().st_mtime <= path.stat().st_mtime for p in sources)


def up_to_date() -> bool:
    deps = [p for p in CSRC.glob("*") if p != CALLS_SRC] + list(INCLUDE.glob("*.h"))
    return newer(LIB, deps)


def build_calls(force: bool = False) -> pathlib.Path | None:
    """Compile the extension of ``csrc/torch_calls.cpp`` against the installed torch if it is
    not there. The package works without it: what goes wrong is a warning, and None."""
    try:
        import sysconfig

        import torch

        path = calls_path()
        if not force and newer(path, [CALLS_SRC, *INCLUDE.glob("*.h")]):
            return path
        LIBDIR.mkdir(exist_ok=True)
        for old in LIBDIR.glob("_srdit_calls*"):   # of older sources, or of another torch
            old.unlink()
        root = pathlib.Path(torch.__file__).parent
        cuda = pathlib.Path(nvcc_path()).resolve().parents[1]
        tmp = path.with_suffix(".so.tmp")
        includes = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
                    cuda / "include", sysconfig.get_paths()["include"]]
        cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared",
               f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
               *(x for i in includes for x in ("-isystem", str(i))), str(CALLS_SRC),
               "-o", str(tmp), f"-L{root / 'lib'}", "-ltorch_python", "-lc10", "-lc10_cuda",
               f"-Wl,-rpath,{root / 'lib'}"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        (LIBDIR / "calls.log").write_text(f"$ {' '.join(cmd)}\n{r.stdout}{r.stderr}")
        if r.returncode != 0:
            raise RuntimeError(f"g++ failed for {CALLS_SRC.name}:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, path)
        return path
    except Exception as e:   # no compiler, no headers, another torch's interface: all the same here
        warnings.warn("the extension of torch_calls.cpp was not built, so the wrappers make all of "
                      f"their checks in Python: {e}", RuntimeWarning, stacklevel=2)
        return None


def build(force: bool = False, verbose: bool = False) -> pathlib.Path:
    """Compile the library if any source is newer than it, then the extension. Returns the
    library's path."""
    if force or not up_to_date():
        log = build_library()
        if verbose:
            print(log)
    build_calls(force)
    return LIB


def build_library() -> str:
    """Compile and link the library; the compilers' log."""
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
    os.replace(tmp, LIB)
    log = "\n".join(logs)
    (LIBDIR / "build.log").write_text(log)
    return log


if __name__ == "__main__":
    p = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(p)
