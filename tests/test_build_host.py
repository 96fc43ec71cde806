"""What the build runs and when, with the compilers replaced by a fake that writes its output file."""
import importlib.util
import os
import subprocess
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(tmp_path, monkeypatch):
    """The build module with its outputs under tmp_path; ``build.ran`` lists the commands."""
    spec = importlib.util.spec_from_file_location("tts_build", os.path.join(REPO, "tt-splat_b200", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    fake = tmp_path / "nvcc"
    fake.write_text("")
    monkeypatch.setenv("NVCC", str(fake))
    for name, file in (("BUILD", "obj"), ("LIB", "lib.so"), ("TORCH_OPS", "ops.so")):
        monkeypatch.setattr(mod, name, str(tmp_path / file))
    mod.ran, mod.rc = [], 0

    def run(cmd, **_):
        mod.ran.append(cmd)
        if mod.rc == 0:
            with open(cmd[cmd.index("-o") + 1], "w") as f:
                f.write(" ".join(cmd))
        return subprocess.CompletedProcess(cmd, mod.rc, "", "")

    monkeypatch.setattr(mod.subprocess, "run", run)
    return mod


def test_the_library_needs_no_torch(build, monkeypatch, capsys):
    """Every C source and the link run through nvcc with torch not importable and no torch function built."""
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build_library(verbose=False) == build.LIB and os.path.exists(build.LIB)
    assert len(build.ran) == len(build._sources()) + 1
    assert all(os.path.basename(c[0]) == "nvcc" for c in build.ran) and not os.path.exists(build.TORCH_OPS)
    assert build.build_all() == build.LIB and "without the torch functions" in capsys.readouterr().out


def test_the_whole_build_has_the_torch_functions(build):
    build.build_all(verbose=False)
    assert os.path.exists(build.LIB) and os.path.exists(build.TORCH_OPS)
    n = len(build.ran)
    build.build_all(verbose=False)
    assert len(build.ran) == n                     # nothing is newer


def test_torch_functions_follow_what_they_are_built_against(build, monkeypatch):
    """Another torch, Python or command rebuilds them; a build that fails leaves the old file, and the next one
    tries again."""
    import torch
    build.build_torch_ops(verbose=False)
    assert len(build.ran) == 1
    build.build_torch_ops(verbose=False)
    assert len(build.ran) == 1
    changes = [(torch, "__version__", "9.9.9"), (sys, "version", "3.99"),
               (build, "_torch_ops_command", lambda old=build._torch_ops_command: old() + ["-DOTHER"])]
    for n, (obj, name, value) in enumerate(changes):
        monkeypatch.setattr(obj, name, value)
        build.build_torch_ops(verbose=False)
        assert len(build.ran) == n + 2
        build.build_torch_ops(verbose=False)
        assert len(build.ran) == n + 2
    with open(build.TORCH_OPS) as f:
        old = f.read()
    monkeypatch.setattr(torch, "__version__", "9.9.10")
    build.rc = 1
    for n in (5, 6):
        with pytest.raises(RuntimeError, match="torch_ops.cpp"):
            build.build_torch_ops(verbose=False)
        assert len(build.ran) == n
        with open(build.TORCH_OPS) as f:
            assert f.read() == old
    build.rc = 0
    build.build_torch_ops(verbose=False)
    assert len(build.ran) == 7
