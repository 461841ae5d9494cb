"""Copies of a ``TokenOrder`` (deepcopy, pickle) own their tables: nothing in them names the original's memory."""
import copy
import pickle

import pytest
import torch

import fused_moe_b200 as F

COPIES = {"deepcopy": copy.deepcopy, "pickle": lambda o: pickle.loads(pickle.dumps(o))}


@pytest.mark.parametrize("how", COPIES)
def test_addresses_are_those_of_the_copys_own_table(how):
    order = F.TokenOrder(torch.device("cpu"), 5, 3, 32, 7, 2, 16)
    order._table.copy_(torch.arange(order._table.numel(), dtype=torch.int32))
    other = COPIES[how](order)
    assert other._table.data_ptr() != order._table.data_ptr()
    assert other._pointers == (other.pos.data_ptr(), other.pair.data_ptr(), other.offsets.data_ptr())
    for name in ("pos", "pair", "offsets", "counts"):
        assert torch.equal(getattr(other, name), getattr(order, name))
    for name in ("tokens", "top_k", "rows", "e_local", "local_expert_offset", "align", "device"):
        assert getattr(other, name) == getattr(order, name)


@pytest.mark.gpu
@pytest.mark.parametrize("how", COPIES)
def test_a_copy_outlives_the_original(how):
    """The original's memory is zeroed (every index in range) and kept before the copy is used."""
    dev = torch.device("cuda", 0)
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 12, (70, 4), generator=g).to(dev)
    x = torch.randn(70, 96, generator=g).to(dev).requires_grad_(True)
    w = torch.rand(70, 4, generator=g).to(dev).requires_grad_(True)

    def use(o):
        rows = F.permute(x, o)
        out = F.unpermute(rows, o, w)
        return (rows, out) + torch.autograd.grad(out.square().sum(), (x, w))
    order = F.sort_tokens(ids, 10, 1, align=8)
    want = use(order)
    other = COPIES[how](order)
    order._table.zero_()
    held = order._table
    del order
    for a, b in zip(use(other), want):
        assert torch.equal(a, b)
    assert not held.any()
