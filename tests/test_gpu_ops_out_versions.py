"""``out=`` is a change that autograd sees: what a graph saved cannot be overwritten unnoticed."""
import pytest
import torch

import fused_moe_b200 as F
from fused_moe_b200 import ops

DEV = "cuda:0"
OVERWRITTEN = pytest.raises(RuntimeError, match="modified by an inplace operation")


def test_the_version_is_counted_without_a_gpu():
    t = torch.zeros(4, 4)
    part = t[1:3]
    ops._written(part)
    assert t._version == 1 and part._version == 1
    with torch.inference_mode():
        ops._written(torch.zeros(2))


@pytest.mark.gpu
def test_a_saved_tensor_that_is_written_into():
    g = torch.Generator(device=DEV).manual_seed(0)
    T, H, K, E = 12, 32, 2, 4
    order = F.sort_tokens(torch.randint(0, E, (T, K), generator=g, device=DEV), E)
    x = torch.randn(T, H, generator=g, device=DEV)
    w = torch.rand(T, K, generator=g, device=DEV).requires_grad_(True)
    y = F.permute(x, order)
    out = F.unpermute(y, order, w)                         # saves y for the gradient of w
    want = torch.autograd.grad(out.sum(), w)[0]
    out = F.unpermute(y, order, w)
    F.permute(2 * x, order, out=y)
    with OVERWRITTEN:
        torch.autograd.grad(out.sum(), w)
    out = F.unpermute(y, order, w)                         # a graph made afterwards is fine
    assert torch.equal(torch.autograd.grad(out.sum(), w)[0], 2 * want)

    s = torch.rand(T, H, generator=g, device=DEV)
    leaf = torch.rand(T, H, generator=g, device=DEV).requires_grad_(True)
    prod = leaf * s
    with torch.no_grad():
        F.unpermute(y, order, w, out=s)
    with OVERWRITTEN:
        torch.autograd.grad(prod.sum(), leaf)

    codes, scale = F.quantize(torch.randn(T, H, generator=g, device=DEV))
    r = torch.rand(T, T + 4, generator=g, device=DEV)
    leaf = torch.rand(T, T + 4, generator=g, device=DEV).requires_grad_(True)
    prod = leaf * r
    F.block_matmul(codes, scale, codes, torch.ones(1, 1, device=DEV), out=r[:, 2:T + 2])   # a part of it
    with OVERWRITTEN:
        torch.autograd.grad(prod.sum(), leaf)
