"""``sort_tokens``, ``permute``, ``unpermute`` and their gradients against plain indexing in 64 bits."""
import numpy as np
import pytest
import torch

import fused_moe_b200 as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}      # half a step below fp16's normal range


def plain_sort(ids, e_local, off, align):
    ids = ids.cpu().numpy().astype(np.int64)
    T, K = ids.shape
    flat = ids.reshape(-1) - off
    lists = [np.nonzero(flat == e)[0] for e in range(e_local)]
    counts = np.array([len(x) for x in lists])
    padded = -(-counts // align) * align
    offsets = np.concatenate([[0], np.cumsum(padded)])
    pairs = T * K
    rows = -(-(pairs + (align - 1) * min(pairs, e_local)) // align) * align
    pair = np.full(rows, -1)
    pos = np.full(pairs, -1)
    for e, x in enumerate(lists):
        pair[offsets[e]:offsets[e] + len(x)] = x
        pos[x] = offsets[e] + np.arange(len(x))
    return offsets, counts, pos.reshape(T, K), pair


def random_ids(T, K, experts, seed, dtype=torch.int32, skew=1.0):
    g = torch.Generator().manual_seed(seed)
    liked = torch.randn(T, experts, generator=g) + skew * torch.randn(experts, generator=g)
    if K <= experts:
        return torch.topk(liked, K, 1).indices.to(dtype).to(DEV)
    return torch.randint(0, experts, (T, K), generator=g).to(dtype).to(DEV)


def check_order(order, ids, e_local, off, align):
    want = plain_sort(ids, e_local, off, align)
    for name, w in zip(("offsets", "counts", "pos", "pair"), want):
        got = getattr(order, name)
        assert got.dtype == torch.int32
        np.testing.assert_array_equal(got.cpu().numpy(), w, err_msg=name)


@pytest.mark.parametrize("T,K,experts,e_local,off,align", [
    (1, 1, 1, 1, 0, 1), (1, 8, 256, 256, 0, 128), (5, 2, 4, 4, 0, 16), (16, 8, 256, 32, 64, 1), (33, 6, 160, 160, 0, 1),
    (100, 32, 64, 64, 0, 7), (129, 8, 256, 1, 255, 128), (400, 3, 1024, 1024, 0, 1), (1000, 8, 300, 257, 20, 128),
    (1023, 8, 256, 256, 0, 128), (1025, 8, 256, 256, 0, 1), (5000, 4, 700, 700, 0, 4), (9001, 8, 64, 64, 0, 1),
    (12000, 5, 1024, 1024, 0, 16), (100000, 7, 40, 33, 5, 1), (70000, 8, 256, 256, 0, 128), (200001, 1, 1000, 900, 50, 1)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_sort(T, K, experts, e_local, off, align, dtype):
    ids = random_ids(T, K, experts, T + K, dtype)
    check_order(F.sort_tokens(ids, e_local, off, align=align), ids, e_local, off, align)


@pytest.mark.parametrize("T", [300, 3000])
def test_sort_of_odd_choices(T):
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(-5, 40, (T, 6), generator=g)                   # out of range on both sides, experts named twice
    ids[0] = torch.tensor([2 ** 62, -2 ** 63, 2 ** 63 - 1, -1, 3, 3])
    ids = ids.to(DEV)
    check_order(F.sort_tokens(ids, 20, 10, align=8), ids, 20, 10, 8)
    check_order(F.sort_tokens(ids.clamp(-5, 40).int(), 32, 0), ids.clamp(-5, 40), 32, 0, 1)
    one = torch.full((T, 6), 3, dtype=torch.int32, device=DEV)         # all on one expert, and none anywhere
    check_order(F.sort_tokens(one, 8, 0, align=128), one, 8, 0, 128)
    check_order(F.sort_tokens(one, 8, 4, align=128), one, 8, 4, 128)
    wide = torch.randint(0, 16, (T, 11), generator=g).to(DEV)
    check_order(F.sort_tokens(wide[:, 2:6], 16), wide[:, 2:6], 16, 0, 1)
    check_order(F.sort_tokens(wide.t().contiguous().t(), 16), wide, 16, 0, 1)
    check_order(F.sort_tokens(wide[:0], 16, align=4), wide[:0], 16, 0, 4)


@pytest.mark.parametrize("dtype", TYPES + [torch.uint8, torch.float8_e4m3fn, torch.int32])
@pytest.mark.parametrize("T,H,K,e_local,align", [(1, 7168, 8, 256, 1), (7, 1, 2, 16, 4), (50, 129, 8, 64, 16), (301, 520, 6, 8, 128)])
def test_permute(dtype, T, H, K, e_local, align):
    ids = random_ids(T, K, 64 if e_local < 256 else 256, H)
    order = F.sort_tokens(ids, e_local, align=align)
    g = torch.Generator().manual_seed(T)
    x = torch.randint(1, 100, (T, H), generator=g).to(torch.float32).to(dtype).to(DEV)
    pair = order.pair.long()
    want = torch.where((pair >= 0)[:, None], x.float()[pair.clamp_min(0) // K], 0.0)
    assert torch.equal(F.permute(x, order).float(), want)
    wide = torch.zeros(T, H + 7, dtype=dtype, device=DEV)
    wide[:, 3:3 + H] = x
    assert torch.equal(F.permute(wide[:, 3:3 + H], order).float(), want)
    # a tensor of the caller's: padding is zeroed, rows behind the last segment and columns beside stay as they were
    host = torch.full((order.rows, H + 16), 80.0, device=DEV).to(dtype)
    F.permute(x, order, out=host[:, 16 // x.element_size():][:, :H])
    used, at = int(order.offsets[-1]), 16 // x.element_size()
    assert torch.equal(host[:used, at:at + H].float(), want[:used])
    assert (host[used:].float() == 80).all() and (host[:, :at].float() == 80).all() and (host[:, at + H:].float() == 80).all()


def sums(y, pos, w):
    """(sum_k w y[pos], sum_k |w y[pos]|) in fp64."""
    v = torch.where((pos >= 0)[..., None], y.double()[pos.clamp_min(0).long()], 0.0)
    v = v if w is None else v * torch.where(pos >= 0, w.double(), 0.0)[..., None]
    return v.sum(1), v.abs().sum(1)


SIZES = [(1, 7168, 8, 256, 256, 1), (7, 1, 2, 16, 16, 4), (50, 129, 8, 64, 16, 16), (301, 520, 6, 64, 64, 128), (64, 2048, 32, 40, 40, 1),
         (1200, 72, 1, 8, 8, 1), (10, 1031, 9, 30, 30, 1), (20, 1602, 10, 30, 30, 1), (700, 4097, 8, 64, 64, 1), (3000, 514, 3, 16, 12, 1),
         (5000, 250, 9, 16, 16, 1), (1100, 320, 3, 16, 16, 8)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,K,experts,e_local,align", SIZES)
@pytest.mark.parametrize("weighted", [True, False])
def test_unpermute(dtype, T, H, K, experts, e_local, align, weighted):
    """K fused multiply-adds, each half an ulp of a partial sum: (K + 1) 2^-24 S with S the sum of absolute terms (their own
    growth below the one more), then half an ulp of the result's type."""
    ids = random_ids(T, K, experts, K)
    order = F.sort_tokens(ids, e_local, align=align)
    g = torch.Generator(device=DEV).manual_seed(H)
    y = torch.randn(order.rows, H + 3, generator=g, device=DEV).to(dtype)
    w = torch.rand(T, K + 2, generator=g, device=DEV) if weighted else None
    for yv in (y[:, :H].contiguous(), y[:, 3:]):
        wv = w[:, 1:1 + K] if weighted else None
        out = F.unpermute(yv, order, wv)
        ref, mass = sums(yv, order.pos, wv)
        err = (K + 1) * 2.0 ** -24 * mass
        assert ((out.double() - ref).abs() <= err + HALF_ULP[dtype] * (ref.abs() + err) + TINY[dtype]).all()
        host = torch.full((T, H + 5), 7.0, device=DEV, dtype=dtype)
        F.unpermute(yv, order, wv, out=host[:, 2:2 + H])
        assert torch.equal(host[:, 2:2 + H], out) and (host[:, :2] == 7).all() and (host[:, 2 + H:] == 7).all()


def test_choices_that_are_not_local_add_nothing():
    ids = torch.tensor([[0, 9], [9, 8], [1, 0]], device=DEV)
    order = F.sort_tokens(ids, 2)
    y = torch.full((order.rows, 40), float("nan"), device=DEV)         # garbage behind the last segment is never read
    y[:3] = torch.arange(3.0, device=DEV)[:, None] + 1
    w = torch.tensor([[2.0, float("nan")], [float("inf"), float("nan")], [3.0, 4.0]], device=DEV)
    want = torch.tensor([2 * 1.0, 0.0, 3 * 3.0 + 4 * 2.0], device=DEV)[:, None].expand(3, 40)
    assert torch.equal(F.unpermute(y, order, w), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,K,experts,e_local,align", SIZES)
def test_gradients(dtype, T, H, K, experts, e_local, align):
    """dx: K additions. dy: one product. dw: H fused multiply-adds in some order, at most (H + 8) 2^-24 of the absolute terms."""
    ids = random_ids(T, K, experts, K + 1)
    order = F.sort_tokens(ids, e_local, align=align)
    g = torch.Generator(device=DEV).manual_seed(H + 1)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)            # noqa: E731
    x, y = r(T, H).to(dtype).requires_grad_(True), r(order.rows, H).to(dtype).requires_grad_(True)
    w = r(T, K).requires_grad_(True)
    d_rows, d_out = r(order.rows, H + 1).to(dtype)[:, 1:], r(T, H).to(dtype)
    rows, out = F.permute(x, order), F.unpermute(y, order, w)
    dx, dy, dw = torch.autograd.grad((rows, out), (x, y, w), (d_rows, d_out))
    pos, pair = order.pos, order.pair.long()
    ref, mass = sums(d_rows, pos, None)
    err = (K + 1) * 2.0 ** -24 * mass
    assert ((dx.double() - ref).abs() <= err + HALF_ULP[dtype] * (ref.abs() + err) + TINY[dtype]).all()
    at = pair.clamp_min(0)
    ref = torch.where((pair >= 0)[:, None], w.detach().double().reshape(-1)[at][:, None] * d_out.double()[at // K], 0.0)
    assert ((dy.double() - ref).abs() <= (2.0 ** -23 + HALF_ULP[dtype]) * ref.abs() + TINY[dtype]).all()
    terms = torch.where((pos >= 0)[..., None], y.detach().double()[pos.clamp_min(0).long()] * d_out.double()[:, None], 0.0)
    assert ((dw.double() - terms.sum(-1)).abs() <= (H + 8) * 2.0 ** -24 * terms.abs().sum(-1)).all()
    assert (dw[pos < 0] == 0).all()
    # each gradient alone, and without weights
    out = F.unpermute(y.detach(), order, w)
    assert torch.equal(torch.autograd.grad(out, w, d_out)[0], dw)
    out = F.unpermute(y, order, w.detach())
    assert torch.equal(torch.autograd.grad(out, y, d_out)[0], dy)
    out = F.unpermute(y, order)
    dy1, = torch.autograd.grad(out, y, d_out)
    assert torch.equal(dy1, torch.where((pair >= 0)[:, None], d_out[at // K], torch.zeros((), dtype=dtype, device=DEV)))


def test_gradients_against_differences():
    """The output is linear in x, in y and in w: a difference over any step is the derivative, up to rounding (fp32 values of
    size one, sums of at most 600 terms: well below 2^-12 of the sum of absolute terms)."""
    T, H, K = 30, 20, 4
    order = F.sort_tokens(random_ids(T, K, 10, 3), 8, 1, align=4)
    g = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)            # noqa: E731
    x, w = r(T, H).requires_grad_(True), r(T, K).requires_grad_(True)
    probe = r(T, H)

    def loss(x, w):
        return (F.unpermute(F.permute(x, order) * 1.5, order, w).double() * probe).sum()
    loss(x, w).backward()
    for leaf, step in ((x, r(T, H)), (w, r(T, K))):
        moved = [(t + step if t is leaf else t).detach() for t in (x, w)]
        diff = loss(*moved) - loss(x.detach(), w.detach())
        want = (leaf.grad.double() * step.double()).sum()
        size = (leaf.grad.double() * step.double()).abs().sum() + loss(x.detach().abs(), w.detach().abs()).abs()
        assert abs(diff - want) <= 2.0 ** -12 * size


def test_gradient_of_a_broadcast_row_and_of_an_expanded_gradient():
    T, H, K = 40, 64, 3
    order = F.sort_tokens(random_ids(T, K, 9, 3), 9)
    row = torch.randn(1, H, device=DEV, requires_grad=True)
    F.permute(row.expand(T, H), order).sum().backward()
    assert torch.equal(row.grad, torch.full((1, H), float(T * K), device=DEV))
    y = torch.ones(order.rows, H, device=DEV, requires_grad=True)
    w = torch.ones(T, K, device=DEV, requires_grad=True)
    F.unpermute(y, order, w).sum().backward()                          # the incoming gradient is an expanded one
    assert (y.grad == 1).all() and (w.grad == H).all()
    one = torch.full((), 0.5, device=DEV, requires_grad=True)
    F.unpermute(y.detach(), order, one.expand(T, K)).sum().backward()
    assert float(one.grad) == T * K * H


def test_refusals():
    ids = random_ids(6, 2, 8, 0)
    order = F.sort_tokens(ids, 8)
    x = torch.zeros(6, 32, device=DEV)
    y, w = torch.zeros(order.rows, 32, device=DEV), torch.zeros(6, 2, device=DEV)
    for bad in (dict(e_local=0), dict(e_local=1025), dict(local_expert_offset=-1), dict(align=0), dict(align=65537)):
        with pytest.raises(ValueError):
            F.sort_tokens(ids, **bad)
    with pytest.raises(ValueError):
        F.sort_tokens(torch.zeros(6, 33, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        F.sort_tokens(ids[0])
    with pytest.raises(TypeError):
        F.sort_tokens(ids.float())
    for call in (lambda: F.permute(x[:5], order), lambda: F.permute(x[0], order), lambda: F.unpermute(y[:-1], order),
                 lambda: F.unpermute(y, order, w[:, :1]), lambda: F.permute(x, order, out=y[:-1]),
                 lambda: F.unpermute(y, order, w, out=torch.zeros(32, 6, device=DEV).t())):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: F.permute(x.double(), order), lambda: F.unpermute(y.double(), order), lambda: F.unpermute(y, order, w.half()),
                 lambda: F.unpermute(y.int(), order)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: F.unpermute(y, order, w.cpu()), lambda: F.permute(x.requires_grad_(True), order, out=y),
                 lambda: F.unpermute(y, order, w.requires_grad_(True), out=torch.zeros(6, 32, device=DEV))):
        with pytest.raises(RuntimeError):
            call()
