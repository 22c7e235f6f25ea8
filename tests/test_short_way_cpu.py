"""The extension that is a short way from torch tensors to the C entries: the package builds and
works without it."""
import pathlib
import subprocess

import pytest
import torch


@pytest.fixture
def built(srdit, tmp_path, monkeypatch):
    """build.py with its outputs in a folder of its own, and compilers that write a line."""
    build = srdit._lib.build
    monkeypatch.setattr(build, "LIBDIR", tmp_path)
    monkeypatch.setattr(build, "LIB", tmp_path / "libsrdit_b200.so")
    ran = []

    def run(cmd, **kw):
        ran.append(pathlib.Path(cmd[0]).name)
        if ran[-1] == "g++" and built.fails is not None:
            raise built.fails
        pathlib.Path(cmd[cmd.index("-o") + 1]).write_text(f"of {len(ran)}")
        return subprocess.CompletedProcess(cmd, built.code if ran[-1] == "g++" else 0, "", "no")

    def built():
        del ran[:]
        build.build()
        return list(ran)

    built.fails, built.code = None, 0
    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "nvcc_path", lambda: "/usr/local/cuda/bin/nvcc")
    built.module, built.folder = build, tmp_path
    return built


def test_builds_once(built):
    ran = built()
    assert ran.count("g++") == 1 and "nvcc" in ran
    assert built.module.LIB.exists() and built.module.calls_path().exists()
    assert built() == []


@pytest.mark.parametrize("fails", (FileNotFoundError("g++"), None))
def test_the_library_is_there_without_a_compiler_of_the_extension(built, fails):
    built.fails, built.code = fails, 1
    with pytest.warns(RuntimeWarning, match="checks in Python"):
        built()
    assert built.module.LIB.exists() and not built.module.calls_path().exists()
    assert built.module.up_to_date()
    built.fails, built.code = None, 0
    assert built() == ["g++"]       # the library is not compiled again
    assert built.module.calls_path().exists()


def test_an_extension_that_no_longer_builds_is_not_left(built):
    built()
    built.module.calls_path().touch()
    import os
    os.utime(built.module.calls_path(), (1, 1))   # older than its source
    built.code = 1
    with pytest.warns(RuntimeWarning):
        built()
    assert not built.module.calls_path().exists()


def test_another_torch_is_another_extension(srdit, built, monkeypatch):
    built()
    old = built.module.calls_path()
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    assert srdit._lib.calls() is None             # the old one is not loaded
    assert built() == ["g++"]
    assert built.module.calls_path().exists() and not old.exists()


@pytest.mark.parametrize("content", (b"", b"\x7fELF not a library"))
def test_an_extension_that_does_not_load(srdit, tmp_path, monkeypatch, content):
    path = tmp_path / "_srdit_calls.so"
    path.write_bytes(content)
    monkeypatch.setattr(srdit._lib.build, "calls_path", lambda: path)
    with pytest.warns(RuntimeWarning, match="does not load"):
        assert srdit._lib.calls() is None
    # a call then makes its own checks, and says what is wrong
    monkeypatch.setattr(srdit.ops, "_calls", ())
    x = torch.zeros(2, 1, 16, dtype=torch.bfloat16)
    with pytest.warns(RuntimeWarning), pytest.raises(srdit._lib.SrditError, match="CUDA"):
        srdit.ops.packed_attn(x, x, x, torch.tensor([0, 2], dtype=torch.int32))
    assert srdit.ops._calls is None
