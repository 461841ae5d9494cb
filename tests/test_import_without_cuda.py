"""The package imports where torch was built without CUDA (its synthetic inputs and checks run there); calls refuse CPU tensors."""
import subprocess
import sys

from conftest import ROOT

CODE = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
import fused_moe_b200 as F
from fused_moe_b200 import synth
codes, scale = synth.quant_rows_1x128(torch.randn(3, 256))
assert codes.shape == (3, 256)
for call in (lambda: F.quantize(torch.randn(3, 256)), lambda: F.sort_tokens(torch.zeros(3, 8, dtype=torch.int32))):
    try:
        call()
    except RuntimeError as e:
        assert "CUDA tensors only" in str(e)
    else:
        raise SystemExit("a CPU tensor was taken")
"""


def test_import_and_refusals():
    run = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
