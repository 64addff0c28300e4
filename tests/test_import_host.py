"""CPU: the package and its argument checks need nothing that a torch without CUDA lacks."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CODE = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_get")]:
    delattr(torch._C, name)
import muxi_race_b200 as m
import muxi_race_b200.torch_ops
for call in (lambda x: m.add_rms_norm(x, x[0]), lambda x: m.route_topk(x, 2), lambda x: m.quantize_w4(x),
             lambda x: m.add_rms_norm_quant(x, x[0])):
    try:
        call(torch.zeros(4, 64, dtype=torch.float16))
    except ValueError as e:
        assert "CUDA" in str(e), e
    else:
        raise AssertionError("a CPU tensor was accepted")
print("imported")
"""


def test_import_with_a_torch_that_lacks_cuda():
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "imported" in r.stdout, r.stderr[-2000:]
