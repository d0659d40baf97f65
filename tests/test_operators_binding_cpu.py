"""The native entry of the stand-alone operators: what works without it, and when it is built again."""
import subprocess
import sys
from pathlib import Path

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
