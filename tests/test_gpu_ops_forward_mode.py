"""Dual numbers (``torch.autograd.forward_ad``): the operators have no forward-mode derivative and say so.  A dual tensor does not
require a gradient, so nothing else would stop a call from returning a result without its tangent."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

import fused_moe_b200 as F
from fused_moe_b200 import ops

DEV = "cuda:0"
REFUSED = pytest.raises(RuntimeError, match="no forward-mode derivative")


def test_what_is_refused_without_a_gpu():
    x = torch.randn(3, 4)
    with fwad.dual_level():
        dual = fwad.make_dual(x, torch.ones_like(x))
        assert not dual.requires_grad
        ops._refuse_duals("f", x, None, dual.detach())
        with REFUSED:
            ops._refuse_duals("f", x, dual)
        with REFUSED:
            ops._refuse_duals("f", dual[:2])
    assert torch.autograd.forward_ad._current_level < 0     # what the calls look at outside of a level


@pytest.fixture(scope="module")
def setup():
    ids = torch.tensor([[0, 2], [1, 2], [3, 0]], device=DEV)
    order = F.sort_tokens(ids, 4)
    return order, torch.randn(3, 64, device=DEV), torch.randn(order.rows, 64, device=DEV), torch.rand(3, 2, device=DEV)


def dual(t):
    return fwad.make_dual(t, torch.ones_like(t))


@pytest.mark.gpu
@pytest.mark.parametrize("leaf", [False, True])
def test_arguments(setup, leaf):
    order, x, y, w = (t.clone().requires_grad_(leaf) if isinstance(t, torch.Tensor) else t for t in setup)
    with fwad.dual_level(), torch.set_grad_enabled(leaf):
        for call in (lambda: F.permute(dual(x), order), lambda: F.unpermute(dual(y), order), lambda: F.unpermute(y, order, dual(w)),
                     lambda: F.unpermute(dual(y), order, w)):
            with REFUSED:
                call()
        # tensors without a tangent are used as ever
        assert torch.equal(F.permute(x, order), F.permute(dual(x).detach(), order))


@pytest.mark.gpu
def test_arguments_of_what_has_no_gradient_at_all(setup):
    x = setup[1]
    codes, scale = F.quantize(x)
    with fwad.dual_level():
        with REFUSED:
            F.quantize(dual(x))
        for args in ((codes, dual(scale), codes, torch.ones(1, 1, device=DEV)), (codes, scale, codes, dual(torch.ones(1, 1, device=DEV)))):
            with REFUSED:
                F.block_matmul(*args)


@pytest.mark.gpu
def test_results_written_into_a_dual(setup):
    order, x, y, w = setup
    codes, scale = F.quantize(x)
    one = torch.ones(1, 1, device=DEV)
    with fwad.dual_level():
        with REFUSED:
            F.permute(x, order, out=dual(torch.empty_like(y)))
        with REFUSED:
            F.unpermute(y, order, w, out=dual(torch.empty_like(x)))
        with REFUSED:
            F.block_matmul(codes, scale, codes, one, out=dual(torch.empty(3, 3, device=DEV)))


@pytest.mark.gpu
def test_gradients_that_are_dual(setup):
    order, x, y, w = setup
    for call, leaf in ((lambda t: F.permute(t, order), x), (lambda t: F.unpermute(t, order, w), y), (lambda t: F.unpermute(y, order, t), w)):
        t = leaf.clone().requires_grad_(True)
        out = call(t)
        with fwad.dual_level():
            with REFUSED:
                torch.autograd.grad(out, t, dual(torch.ones_like(out)), retain_graph=True)
        torch.autograd.grad(out, t, torch.ones_like(out))


@pytest.mark.gpu
def test_function_transforms_are_refused_too(setup):
    order, x, y, w = setup
    for call, arg in ((lambda t: F.permute(t, order), x), (lambda t: F.unpermute(t, order, w), y), (lambda t: F.quantize(t)[1], x)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (arg,), (torch.ones_like(arg),))
