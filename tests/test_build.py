"""CPU tests of the build recipe: what is built from what, and what a failure
leaves.  No compiler is run."""

import os
import subprocess

import pytest

from decode_opt_b200 import build as dg_build


class Compilers:
    """Stands in for subprocess.run: notes the outputs asked for, makes them
    (empty files), and fails for those named."""

    def __init__(self, failing=()):
        self.made, self.failing = [], failing

    def __call__(self, cmd, check=False, **kw):
        out = cmd[cmd.index("-o") + 1]
        name = os.path.basename(out).removesuffix(".tmp")
        self.made.append(name)
        if name in self.failing:
            raise subprocess.CalledProcessError(1, cmd)
        open(out, "wb").close()
        return subprocess.CompletedProcess(cmd, 0)


@pytest.fixture
def place(tmp_path, monkeypatch):
    """The build's outputs in a folder of their own."""
    for name in ("LIB_PATH", "HOST_LIB", "DROP_IN_BIN", "CUBLASLT_BIN"):
        monkeypatch.setattr(dg_build, name, str(tmp_path / os.path.basename(getattr(dg_build, name))))
    return tmp_path


@pytest.mark.parametrize("force", [False, True])
def test_the_library_needs_no_torch(place, monkeypatch, force):
    """A host compiler that refuses torch's headers, or no torch at all: the C
    library is built all the same, and no extension module of before is left
    beside it."""
    run = Compilers(failing=("_host.so",))
    monkeypatch.setattr(subprocess, "run", run)
    (place / "_host.so").write_bytes(b"of another build")
    os.utime(place / "_host.so", (1, 1))
    assert dg_build.build_library(force=force) == dg_build.LIB_PATH
    assert run.made[0] == "libdecode_gemm_b200.so" and os.path.exists(dg_build.LIB_PATH)
    assert not os.path.exists(dg_build.HOST_LIB)
    # The whole build says so.
    with pytest.raises(subprocess.CalledProcessError):
        dg_build.build(force=force)
    monkeypatch.setitem(__import__("sys").modules, "torch", None)
    assert dg_build.build_library(force=True) == dg_build.LIB_PATH
    with pytest.raises(ImportError):
        dg_build.build(force=True)


def test_host_code_does_not_recompile_the_kernels(place, monkeypatch):
    run = Compilers()
    monkeypatch.setattr(subprocess, "run", run)
    dg_build.build()
    assert sorted(run.made) == ["_host.so", "dg_cublaslt_fp8", "dg_drop_in_check", "libdecode_gemm_b200.so"]
    real = os.path.getmtime
    ahead = set()
    monkeypatch.setattr(os.path, "getmtime", lambda p: real(p) + 10 ** 6 * (str(p) in ahead))
    ahead.add(dg_build.HOST_SRC)
    assert not dg_build.needs_build(dg_build.LIB_PATH)
    for source in dg_build.SOURCES + ("sm100.cuh", "warp_mma.cuh"):
        ahead.clear()
        ahead.add(os.path.join(dg_build.CSRC, source))
        assert dg_build.needs_build(dg_build.LIB_PATH), source
    ahead.clear()
    ahead.add(os.path.join(dg_build.INCLUDE, "decode_attention_b200.h"))
    assert dg_build.needs_build(dg_build.LIB_PATH)


def test_another_torch_means_another_extension(place, monkeypatch):
    import torch
    host = place / "_host.so"
    assert dg_build.host_needs_build()
    host.write_bytes(b"code" + dg_build.host_built_for().encode() + b"\0more code")
    assert not dg_build.host_needs_build()
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".1")
    assert dg_build.host_needs_build()
    run = Compilers()
    monkeypatch.setattr(subprocess, "run", run)
    dg_build.build_host()
    assert run.made == ["_host.so"]


def test_the_extension_says_what_it_was_built_for():
    """(In a process of its own: it loads torch's libraries.)"""
    import sys
    code = ("import decode_opt_b200.attention as a, decode_opt_b200.build as b; "
            "print(a._host.built_for == b.host_built_for(), b.host_needs_build())")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=dg_build.ROOT)
    assert out.stdout.split() == ["True", "False"], out.stderr
    # ... and another torch does not run it.
    code = ("import torch; torch.__version__ = '0.0.1'\n"
            "try: import decode_opt_b200.attention\n"
            "except RuntimeError as e: print('build it again' in str(e))")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=dg_build.ROOT)
    assert out.stdout.split() == ["True"], out.stderr
