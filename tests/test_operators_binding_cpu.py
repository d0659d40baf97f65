"""The native entry of the stand-alone operators: what works without it, and when it is built again."""
import importlib.util
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]

WITHOUT = """
import sys
sys.modules["sparsemoe_b200._operators"] = None      # as a binary that does not load
import torch
import sparsemoe_b200 as sm
from sparsemoe_b200.ep import ExpertParallelLayer
assert sm.capacity(512, 2, 8, 1.25) == 160 and sm.MoeLayer and sm.lib.moe_solve_v2 and sm.Routing().struct().scale == 1.0
assert sm.int8_weight(torch.ones(5, 7, dtype=torch.int8)).stride() == (16, 1)
w = torch.zeros(16, 16, dtype=torch.int8)
for call in (lambda: sm.route_experts(torch.zeros(4, 8), 2), lambda: sm.quantize_int8_tokens(torch.zeros(4, 8)),
             lambda: sm.int8_linear(torch.zeros(4, 16), w, torch.ones(16))):
    try:
        call()
    except ImportError as e:
        assert "build.py" in str(e) and "_operators.so" in str(e)
    else:
        raise AssertionError("no error")
print("ok")
"""


def test_the_package_without_the_native_entry():
    r = subprocess.run([sys.executable, "-c", WITHOUT], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


@pytest.fixture
def builder(tmp_path, monkeypatch):
    """sparsemoe_b200/build.py with its outputs under tmp_path and a compiler that writes an empty file."""
    spec = importlib.util.spec_from_file_location("_sm_build_test", ROOT / "sparsemoe_b200" / "build.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    monkeypatch.setattr(mod, "BUILD", tmp_path)
    monkeypatch.setattr(mod, "BINDING", tmp_path / "_operators.so")
    mod.calls = []

    def run(cmd, **kw):
        mod.calls.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).touch()
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(mod.subprocess, "run", run)
    return mod


def test_another_torch_builds_the_entry_again(builder, monkeypatch):
    for _ in range(2):                       # built once
        assert builder.build_binding() == builder.BINDING
    assert len(builder.calls) == 1
    monkeypatch.setattr(builder, "binding_stamp", lambda: "torch 0.0, python 3.0")
    builder.build_binding()
    builder.build_binding()
    assert len(builder.calls) == 2
    (builder.BUILD / "_operators.so.stamp").unlink()      # a binary of unknown origin
    builder.build_binding()
    assert len(builder.calls) == 3


def test_the_stamp_names_torch_and_python(builder):
    import torch
    assert torch.__version__ in builder.binding_stamp() and f"{sys.version_info[0]}.{sys.version_info[1]}" in builder.binding_stamp()


def test_the_library_builds_without_torch(builder, monkeypatch):
    real = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else real(name, *a))
    assert builder.build_binding() is None and not builder.calls
