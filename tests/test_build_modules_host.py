"""The optional host modules: left out where they cannot be built or belong to another torch, never in the way."""

import importlib.util
import os
import subprocess
import types

import pytest
import torch

from kohakufa_cute import native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build(monkeypatch, tmp_path):
    """build.py with its outputs in a folder of their own."""
    spec = importlib.util.spec_from_file_location("kfa_build", os.path.join(ROOT, "kohakufa-cute_b200", "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "OUT_DIR", str(tmp_path))
    monkeypatch.setattr(module, "OBJ_DIR", str(tmp_path))
    return module


def stale(build, name):
    """A module of other sources in the place of the one to be built."""
    path = os.path.join(build.OUT_DIR, name + build.sysconfig.get_config_var("EXT_SUFFIX"))
    with open(path, "w") as f:
        f.write("of other sources")
    return path


MODULES = (("build_records", "_fast_records"), ("build_calls", "_fast_calls"))


@pytest.mark.parametrize("step, name", MODULES)
@pytest.mark.parametrize("error", (OSError("no such compiler"), subprocess.CalledProcessError(1, "cc")))
def test_a_failing_compiler_leaves_a_module_out(build, monkeypatch, step, name, error):
    def failing(*arguments, **keywords):
        raise error

    path = stale(build, name)
    monkeypatch.setattr(build.subprocess, "check_call", failing)
    assert getattr(build, step)(verbose=False) is None and not os.path.exists(path)


@pytest.mark.parametrize("step, name", MODULES)
def test_missing_headers_leave_a_module_out(build, monkeypatch, step, name):
    path = stale(build, name)
    exists = os.path.exists
    monkeypatch.setattr(build.os.path, "exists", lambda p: not str(p).endswith("Python.h") and exists(p))
    monkeypatch.setattr(build.subprocess, "check_call", lambda *a, **k: pytest.fail("compiled without headers"))
    assert getattr(build, step)(verbose=False) is None and not exists(path)


def test_a_module_of_another_torch_is_not_used():
    mine = types.SimpleNamespace(torch_version=str(torch.__version__))
    assert native._of_this_torch(mine) is mine
    for other in (None, types.SimpleNamespace(), types.SimpleNamespace(torch_version="1.0.0")):
        assert native._of_this_torch(other) is None
    if native._fast_calls is not None:
        assert native.fast is native._fast_calls and native.fast.torch_version == str(torch.__version__)
