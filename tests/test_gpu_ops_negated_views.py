"""Views that torch keeps with the other sign (the imaginary part of a conjugate): read by value, refused as a result."""
import pytest
import torch

import fused_moe_b200 as F
from fused_moe_b200 import ops

DEV = "cuda:0"


def negated(t):
    """A [rows, 1] tensor equal to ``t`` whose memory holds ``-t``."""
    z = torch.zeros(t.shape + (2,), dtype=t.dtype, device=t.device)
    z[..., 1] = -t
    v = torch.view_as_complex(z).conj().imag
    assert v.is_neg() and torch.equal(v.resolve_neg(), t)
    return v


def test_a_matrix_is_read_by_value_without_a_gpu():
    t = torch.randn(5, 1)
    for v in (negated(t), negated(t[:1]), negated(torch.randn(3, 4))):
        m, rows, cols, pitch = ops._matrix(v, "t")
        assert not m.is_neg() and (rows, cols) == tuple(v.shape) and pitch == cols
        assert torch.equal(torch.frombuffer(bytearray(m.contiguous().numpy().tobytes()), dtype=torch.float32).view(rows, cols), v.resolve_neg())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_operators_by_value(dtype):
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(40, 1, generator=g, device=DEV).to(dtype)
    ids = torch.randint(0, 6, (40, 1), generator=g, device=DEV)
    order = F.sort_tokens(ids, 6)
    w = torch.rand(40, 1, generator=g, device=DEV)
    for a, b in zip(F.quantize(negated(x)), F.quantize(x)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(F.permute(negated(x), order), F.permute(x, order))
    y = F.permute(x, order)
    assert torch.equal(F.unpermute(negated(y), order, negated(w)), F.unpermute(y, order, w))
    # gradients that arrive so
    lx, ly, lw = x.clone().requires_grad_(True), y.clone().requires_grad_(True), w.clone().requires_grad_(True)
    out = F.unpermute(ly, order, lw)
    for a, b in zip(torch.autograd.grad(out, (ly, lw), negated(x), retain_graph=True), torch.autograd.grad(out, (ly, lw), x)):
        assert torch.equal(a, b)
    rows = F.permute(lx, order)
    for a, b in zip(torch.autograd.grad(rows, lx, negated(y), retain_graph=True), torch.autograd.grad(rows, lx, y)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_scales_by_value():
    a = torch.full((5, 128), 0x38, dtype=torch.uint8, device=DEV)
    sa, sb = torch.tensor([[1.0], [2.0], [-3.0], [0.5], [4.0]], device=DEV), torch.tensor([[2.0]], device=DEV)
    want = (128.0 * sa * sb).expand(5, 5)
    for p, q in ((negated(sa), sb), (sa, negated(sb)), (negated(sa), negated(sb))):
        assert torch.equal(F.block_matmul(a, p, a, q, scale_layout="tk", out_dtype=torch.float32), want)


@pytest.mark.gpu
def test_results_are_refused():
    x = torch.randn(4, 1, device=DEV)
    order = F.sort_tokens(torch.zeros(4, 1, dtype=torch.int32, device=DEV), 1)
    a, one = torch.full((4, 16), 0x38, dtype=torch.uint8, device=DEV), torch.ones(1, 4, device=DEV)
    for call in (lambda o: F.permute(x, order, out=o), lambda o: F.unpermute(x, order, out=o),
                 lambda o: F.block_matmul(a, one, a[:1], one[:, :1], out=o)):
        with pytest.raises(ValueError, match="other sign"):
            call(negated(torch.zeros(4, 1, device=DEV)))
