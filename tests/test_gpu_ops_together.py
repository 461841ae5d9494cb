"""The operators beside the layer as they are used: the layer from its parts, a feed-forward layer in 8 bits, captured graphs,
streams, two calls at once, a training step."""
import pytest
import torch

import fused_moe_b200 as F
from fused_moe_b200 import synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def experts_from_parts(rows, order, w1, s1, w2, s2):
    """Sorted bf16 rows through each expert's two products; segments as the host sees them."""
    out = torch.zeros_like(rows)
    bounds, counts = order.offsets.tolist(), order.counts.tolist()
    for e, n in enumerate(counts):
        if n:
            r = slice(bounds[e], bounds[e] + n)
            q, s = F.quantize(rows[r])
            h = F.block_matmul(q, s, w1[e], s1[e], out_dtype=torch.float32)
            q, s = F.quantize(h, swiglu=True)
            F.block_matmul(q, s, w2[e], s2[e], out=out[r])
    return out


@pytest.mark.parametrize("T,align", [(1, 1), (45, 128), (300, 16)])
def test_the_layer_from_its_parts(T, align):
    """route, sort, permute, quantize, two products with a SwiGLU between them, unpermute: the fused layer up to the roundings that
    differ.  Both round activations to e4m3 before the second product, by other scales, each off by at most half a step (2^-4 of
    a value), which the random second matrix passes on in the 2-norm: 2^-3 of the output's norm bounds the difference."""
    inp = synth.make_inputs(T=T, e_local=32, local_expert_offset=64, seed=3, hidden=1024, inter=256).to(DEV)
    want = F.custom_kernel(*inp.args()).clone()
    x = (inp.hidden_states.float() * inp.hidden_states_scale.t().repeat_interleave(128, 1))
    ids, weights = F.route(inp.routing_logits, inp.routing_bias, inp.routed_scaling_factor, 64, 32, 1024, 256)
    order = F.sort_tokens(ids, 32, 64, align=align)
    rows = F.permute(x, order)                       # (fp32: quantising it again gives the very codes)
    y = experts_from_parts(rows, order, inp.gemm1_weights, inp.gemm1_weights_scale, inp.gemm2_weights, inp.gemm2_weights_scale)
    got = F.unpermute(y, order, weights)
    assert (got - want.float()).norm() <= 2.0 ** -3 * want.float().norm()
    none = (order.pos < 0).all(1)
    assert (got[none] == 0).all() and (want[none] == 0).all()


def test_codes_and_their_scales_travel_too():
    """Sorting quantised rows is quantising sorted rows."""
    x = torch.randn(60, 640, device=DEV)
    order = F.sort_tokens(torch.randint(0, 12, (60, 4), device=DEV), 12, align=16)
    q, s = F.quantize(x, scale_layout="tk")
    qr, sr = F.quantize(F.permute(x, order), scale_layout="tk")
    live = order.pair >= 0
    assert torch.equal(F.permute(q, order).view(torch.uint8)[live], qr.view(torch.uint8)[live])
    assert torch.equal(F.permute(s, order)[live], sr[live])


def feed_forward(x, w1, s1, w2, s2):
    q, s = F.quantize(x)
    q, s = F.quantize(F.block_matmul(q, s, w1, s1), swiglu=True)
    return F.block_matmul(q, s, w2, s2)


def weights_for(hidden, inter):
    w1, s1, w2, s2 = synth.make_expert(0, 0, hidden, inter, DEV)
    return w1, s1, w2, s2


@pytest.mark.parametrize("T", [1, 16, 333])
def test_captured_and_replayed(T):
    w = weights_for(1024, 512)
    x = torch.randn(T, 1024, device=DEV, dtype=torch.bfloat16)
    ids = torch.randint(0, 20, (T, 6), device=DEV)
    mix = torch.rand(T, 6, device=DEV)

    def step():
        order = F.sort_tokens(ids, 16, 2, align=8)
        rows = F.permute(x, order)
        return order.pos, rows, F.unpermute(rows, order, mix), feed_forward(x, *w)
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                               # two graphs of the same tensors
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    for seed in range(3):
        x.copy_(torch.randn(T, 1024, generator=torch.Generator().manual_seed(seed)))
        ids.copy_(torch.randint(0, 20, (T, 6), generator=torch.Generator().manual_seed(seed)))
        want = [t.clone() for t in step()]
        streams = [torch.cuda.Stream() for _ in graphs]
        for (g, _), st in zip(graphs, streams):      # replayed side by side
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        for _, res in graphs:
            for a, b in zip(res, want):
                assert torch.equal(a, b)


def test_calls_on_two_streams_at_once():
    w = weights_for(2048, 512)
    xs = [torch.randn(t, 2048, device=DEV, dtype=torch.bfloat16) for t in (3, 150, 40, 700)]
    idss = [torch.randint(0, 64, (20000 + i, 4), device=DEV) for i in range(4)]
    want = [feed_forward(x, *w) for x in xs]
    orders = [F.sort_tokens(i, 64).pos.clone() for i in idss]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        got = []
        for x, i, st in zip(xs, idss, streams):
            with torch.cuda.stream(st):
                got.append((feed_forward(x, *w), F.sort_tokens(i, 64).pos))
        torch.cuda.synchronize()
        for (a, p), b, q in zip(got, want, orders):
            assert torch.equal(a, b) and torch.equal(p, q)


def test_a_training_step_with_experts_between_captured_too():
    """Experts under training between permute and unpermute: gradients of tokens, router weights and expert weights, eager and
    captured with torch.autograd.grad, against plain indexing in 64 bits.  All in fp32: a gradient is a chain of three sums of at
    most 128 terms, each within 128 * 2^-24 of its absolute terms, which random signs leave far below 2^-18 of the norm."""
    T, H, K, E = 64, 128, 2, 4
    g = torch.Generator().manual_seed(0)
    x = torch.randn(T, H, generator=g).to(DEV).requires_grad_(True)
    we = (torch.randn(E, H, H, generator=g) / H ** 0.5).to(DEV).requires_grad_(True)
    mix = torch.rand(T, K, generator=g).to(DEV).requires_grad_(True)
    ids = torch.topk(torch.randn(T, E, generator=g), K, 1).indices.to(DEV)
    counts = torch.bincount(ids.reshape(-1), minlength=E).tolist()
    order = F.sort_tokens(ids, E)
    probe = torch.randn(T, H, generator=g).to(DEV)

    def step():
        rows = F.permute(x, order).split(counts)
        y = torch.cat([r @ we[e] for e, r in enumerate(rows)])
        return torch.autograd.grad((F.unpermute(y, order, mix) * probe).sum(), (x, we, mix))
    eager = step()
    xd, wd, md = (t.detach().double().requires_grad_(True) for t in (x, we, mix))
    out = torch.einsum("tk,tkh->th", md, torch.einsum("th,tkhj->tkj", xd, wd[ids]))
    for a, b in zip(eager, torch.autograd.grad((out * probe.double()).sum(), (xd, wd, md))):
        assert (a.double() - b).norm() <= 2.0 ** -18 * b.norm()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    graph.replay()
    for a, b in zip(captured, eager):
        assert torch.equal(a, b)
    assert torch.equal(step()[0], eager[0])


def test_offsets_beyond_32_bits():
    """Rows behind the 4 GiB mark of every operator's large side, spot-checked where the offset has more than 32 bits."""
    T, H, K = 40960, 7168, 8                         # sorted rows: 4.7 GB of bf16
    ids = torch.arange(T * K, device=DEV).view(T, K) % 16
    order = F.sort_tokens(ids, 16)
    x = torch.arange(T, device=DEV, dtype=torch.float32)[:, None].expand(T, H).bfloat16().contiguous()
    rows = F.permute(x, order)
    tail = order.pair[-1000:].long() // K
    assert torch.equal(rows[-1000:], x[tail])
    out = F.unpermute(rows, order, torch.full((T, K), 0.125, device=DEV))
    assert torch.equal(out, x)
    del out
    y = rows.requires_grad_(True)
    dy, = torch.autograd.grad(F.unpermute(y, order), y, x)
    assert torch.equal(dy[-1000:], x[tail])
    del rows, y, dy
    big = torch.zeros(T, 65536, device=DEV, dtype=torch.bfloat16)    # 5.4 GB of activations, 2.7 GB of codes
    big[-1] = torch.randn(65536, device=DEV)
    q, s = F.quantize(big)
    one, so = F.quantize(big[-1:])
    assert torch.equal(q[-1:].view(torch.uint8), one.view(torch.uint8)) and torch.equal(s[:, -1:], so)
    assert not q[:-1].view(torch.uint8).any()
    del big
    w = torch.zeros(128, 65536, device=DEV, dtype=torch.uint8)
    w[:, ::512] = 0x38                                               # ones
    sw = torch.ones(1, 512, device=DEV)
    small = F.block_matmul(one, so, w, sw, out_dtype=torch.float32)
    wide = torch.empty(T, 32768, device=DEV, dtype=torch.float32)    # 5.4 GB, of which the first 128 columns are the result
    F.block_matmul(q, s, w, sw, out=wide[:, :128])
    ref = (one.double() * so.double().t().repeat_interleave(128, 1))[:, ::512].sum()
    for got in (small[0], wide[-1, :128]):
        assert ((got.double() - ref).abs() <= 2.0 ** -13 * (one.double().abs() * so.double().t().repeat_interleave(128, 1))[:, ::512].sum()).all()
    assert not wide[:-1, :128].any()


def test_second_derivatives_are_refused():
    ids = torch.randint(0, 8, (64, 4), dtype=torch.int32, device=DEV)
    order = F.sort_tokens(ids)
    x = torch.randn(64, 32, device=DEV).requires_grad_(True)
    y = torch.randn(order.rows, 32, device=DEV).requires_grad_(True)
    w = torch.rand(64, 4, device=DEV).requires_grad_(True)
    for out, leaf in ((F.permute(x, order), x), (F.unpermute(y, order, w), y)):
        d = torch.ones_like(out).requires_grad_(True)
        grad, = torch.autograd.grad(out, leaf, d, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            grad.sum().backward()
