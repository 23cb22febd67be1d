"""The short cuts of superkmeans_b200/ops.py are built for one torch and one Python, are not used with others, and are not needed."""
import os
import subprocess
import sys

import pytest
import torch

import __graft_entry__
from superkmeans_b200 import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(tmp_path, monkeypatch):
    """The build script, with its outputs elsewhere."""
    build = __graft_entry__._load_build_module()
    for name in ("CALLS_OUTPUT", "CALLS_BUILT_FOR"):
        monkeypatch.setattr(build, name, str(tmp_path / os.path.basename(getattr(build, name))))
    monkeypatch.setattr(build, "HERE", str(tmp_path))
    return build


def test_those_in_use_were_built_for_what_they_run_with():
    build = __graft_entry__._load_build_module()
    assert ops._calls.built_for == build.calls_built_for(os.path.dirname(torch.__file__))
    assert torch.__version__ in ops._calls.built_for and not build._stale_calls(ops._calls.built_for)


def test_another_torch_makes_them_stale(build):
    assert build._stale_calls("a")
    for path in (build.CALLS_OUTPUT, build.CALLS_BUILT_FOR):
        with open(path, "w") as f:
            f.write("a")
    assert not build._stale_calls("a") and build._stale_calls("b")


def test_a_build_that_cannot_make_them_goes_on(build, monkeypatch, capsys):
    for path in (build.CALLS_OUTPUT, build.CALLS_BUILT_FOR):
        with open(path, "w") as f:
            f.write("of another torch")

    def no_linker(cmd, **_):
        return subprocess.CompletedProcess(cmd, 1, "", "cannot find -lc10_cuda")

    monkeypatch.setattr(build.subprocess, "run", no_linker)
    build.build_calls()
    assert "cannot find -lc10_cuda" in capsys.readouterr().err
    assert not os.path.exists(build.CALLS_OUTPUT) and not os.path.exists(build.CALLS_BUILT_FOR)   # (the old one is not left to be loaded)

    def no_compiler(cmd, **_):
        raise FileNotFoundError("g++")

    monkeypatch.setattr(build.subprocess, "run", no_compiler)
    build.build_calls()
    assert "without its short cuts" in capsys.readouterr().err


@pytest.mark.parametrize("made", ["fake.built_for = 'torch 1.0, CUDA None, cpython-38'", "pass"])
def test_those_of_another_torch_are_left_alone(made):
    code = f"""
import sys, types
fake = types.ModuleType("superkmeans_b200._ops_calls")
fake.lookup = lambda *_: 1 / 0
{made}
sys.modules["superkmeans_b200._ops_calls"] = fake
from superkmeans_b200 import ops
assert ops._calls is not fake and ops._calls.lookup(1, 2) is None and ops._calls.ordinary() is None
print("left alone")
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "left alone" in done.stdout, done.stdout + done.stderr
