"""What becomes of the word that a block_matmul leaves when a bounded wait gave up.  The word is written by the host here: no kernel is
made to fail."""
import os
import subprocess
import sys

import pytest
import torch

import fused_moe_b200 as F
from conftest import ROOT
from fused_moe_b200 import MoEError, _capi, ops

TIMEOUT = -5


def test_refusals_without_a_gpu():
    assert _capi.lib().b200moe_status_words(None) == -1
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        F.check_status("cpu")


def codes(*shape):
    return torch.full(shape, 0x38, dtype=torch.uint8, device="cuda:0")


def product():
    one = torch.ones(1, 1, device="cuda:0")
    return F.block_matmul(codes(1, 128), one, codes(2, 128), one)


@pytest.fixture()
def words():
    product()
    F.check_status()
    st = ops._status[0]
    yield st.view
    st.view[0] = st.view[1] = 0


@pytest.mark.gpu
def test_every_operator_raises_it_once(words):
    ids = torch.tensor([[0, 1], [1, 2]], device="cuda:0")
    order = F.sort_tokens(ids, 4)
    x = torch.randn(2, 64, device="cuda:0")
    rows = F.permute(x, order)
    leaf = x.clone().requires_grad_(True)
    graph = F.permute(leaf, order).sum()
    calls = [product, lambda: F.quantize(x), lambda: F.sort_tokens(ids, 4), lambda: F.permute(x, order),
             lambda: F.unpermute(rows, order), lambda: torch.autograd.grad(graph, leaf, retain_graph=True)]
    for call in calls:
        words[1], words[0] = 7, TIMEOUT
        with pytest.raises(MoEError, match="detail=7") as e:
            call()
        assert e.value.status == TIMEOUT
        call()


@pytest.mark.gpu
@pytest.mark.parametrize("device", [None, 0, "cuda", "cuda:0", torch.device("cuda", 0)])
def test_check_status(words, device):
    words[1], words[0] = 14, TIMEOUT
    with pytest.raises(MoEError, match="detail=14"):
        F.check_status(device)
    F.check_status(device)


@pytest.mark.gpu
def test_the_words_are_the_devices_own(words):
    import ctypes as C
    first, second = C.c_void_p(), C.c_void_p()
    for p in (first, second):
        assert _capi.lib().b200moe_status_words(C.byref(p)) == 0
    assert first.value == second.value == ops._status[0].ptr


FIRST_CALL_CAPTURED = """
import torch, fused_moe_b200 as F
from fused_moe_b200 import ops
torch.zeros(1, device='cuda').add_(1)
a = torch.full((3, 256), 0x38, dtype=torch.uint8, device='cuda')
s = torch.ones(2, 3, device='cuda'); t = torch.ones(1, 2, device='cuda')
seen, call = [], ops._call
def record(name, index, *args):
    seen.append(args[-1]); call(name, index, *args)
ops._call = record
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = F.block_matmul(a, s, a, t, out_dtype=torch.float32)
assert seen == [ops._status[0].ptr] and seen[0], seen
g.replay()
F.check_status()
assert (out == 256).all()
ops._status[0].view[0] = -5
try:
    g.replay(); F.check_status()
except F.MoEError as e:
    assert e.status == -5
else:
    raise SystemExit('a word left after a replay went unseen')
print('ok')
"""


@pytest.mark.gpu
def test_a_first_call_that_is_captured_reports_too():
    run = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout + run.stderr
