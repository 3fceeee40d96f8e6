"""When the tensor binding is built again (no compiler runs)."""
import importlib.metadata
import importlib.util
import os

import pytest
from conftest import PKG


@pytest.fixture
def build(monkeypatch, tmp_path):
    spec = importlib.util.spec_from_file_location("build_native", os.path.join(PKG, "build_native.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    out = tmp_path / "_epq_torch.so"
    monkeypatch.setattr(mod, "OBJ", str(tmp_path / "obj"))
    monkeypatch.setattr(mod, "TORCH_OUT", str(out))
    commands = []

    def compile(cmd):
        commands.append(cmd)
        out.write_bytes(b"")

    monkeypatch.setattr(mod.subprocess, "check_call", compile)
    return lambda **kw: (mod.build_torch(quiet=True, **kw), len(commands))[1]


def test_another_torch_builds_the_binding_again(build, monkeypatch):
    assert build() == 1 and build() == 1
    real = importlib.metadata.version
    monkeypatch.setattr(importlib.metadata, "version", lambda name: "0.0.1" if name == "torch" else real(name))
    assert build() == 2 and build() == 2
    monkeypatch.undo()


def test_force_and_a_missing_file_build_it(build, tmp_path):
    assert build() == 1 and build(force=True) == 2
    (tmp_path / "_epq_torch.so").unlink()
    assert build() == 3 and build() == 3
