"""Workloads of the operators that stand beside the fused layer: quantisation to e4m3 with a scale per 1x128 block, the
block-scaled e4m3 matrix product, and tokens sorted by expert and back (with gradients).

A case is one pass as a user's program makes it; ``run`` computes it with elementary torch operations, or, where ``own``
is true, through ``fused_moe_b200``.  Sizes are the layer's own (hidden 7168, intermediate 2048, 256 experts, top-8) and
generic ones.

Fields of a case:
  op        "quantize", "matmul", "dispatch" (sort + permute), "combine" (sort + unpermute) or "train" (sort, permute,
            unpermute and both gradients)
  tokens    rows of the activations
  dtype     type of the activations; of the result for "matmul"
  quantize: cols (columns of the result), swiglu (the input is [tokens, 2 cols]), layout of the scales ("kt", "tk")
  matmul:   n, k, layout of the activation scales
  tokens sorted: hidden, top_k, experts (of the router), local (held here, from ``offset`` on), align (segments start on
            multiples of it), wide (int64 ids)
"""
import math

import torch

own = False

BLOCK, E4M3_MAX, AMAX_MIN = 128, 448.0, 1e-12
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _quantize(name, tokens, cols, dtype="bf16", swiglu=False, layout="kt"):
    return _named(name, op="quantize", tokens=tokens, cols=cols, dtype=dtype, swiglu=swiglu, layout=layout)


def _matmul(name, tokens, n, k, dtype="bf16", layout="kt"):
    return _named(name, op="matmul", tokens=tokens, n=n, k=k, dtype=dtype, layout=layout)


def _tokens(name, op, tokens, hidden=7168, top_k=8, experts=256, local=256, offset=0, align=1, dtype="bf16", wide=False):
    return _named(name, op=op, tokens=tokens, hidden=hidden, top_k=top_k, experts=experts, local=local, offset=offset,
                  align=align, dtype=dtype, wide=wide)


def _named(name, **case):
    return dict(case, name=name) if name else case


def listed():
    return [
        # activations of a decode step before they enter the layer: a launch's latency
        _quantize("quantize_decode", 4, 7168),
        # a prefill chunk's activations
        _quantize("quantize_prefill", 8192, 7168),
        # between the two products of a feed-forward layer, odd number of rows, scales laid out per token
        _quantize("swiglu_ragged", 4099, 2048, dtype="fp16", swiglu=True, layout="tk"),
        # one token through the always-on expert's gate and up projection: the weights' bytes
        _matmul("matmul_decode", 1, 4096, 7168),
        # a decode batch through its down projection
        _matmul("matmul_batch", 48, 7168, 2048, dtype="fp16"),
        # a short prompt through a projection of odd width, fp32 result
        _matmul("matmul_ragged", 301, 1001, 7168, dtype="fp32", layout="tk"),
        # a prefill chunk through gate and up projection: tensor cores
        _matmul("matmul_prefill", 8192, 4096, 7168),
        # a decode batch sent to its experts
        _tokens("dispatch_decode", "dispatch", 16),
        # a prefill chunk sent to its experts, segments padded to a matrix tile
        _tokens("dispatch_prefill", "dispatch", 4096, align=128),
        # results back to a ragged chunk's tokens on a GPU that holds 32 of the 256 experts
        _tokens("combine_slice", "combine", 901, local=32, offset=64, wide=True),
        # results back to a prefill chunk's tokens
        _tokens("combine_prefill", "combine", 8192),
        # a training step's dispatch and combine, forward and backward, odd number of tokens
        _tokens("train_step", "train", 4097, hidden=2048, experts=64, local=64, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: the kinds of ``listed()`` over their whole ranges."""
    kind = rng.choice(["quantize", "matmul", "matmul", "dispatch", "combine", "train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    layout = rng.choice(["kt", "tk"])
    if kind == "quantize":
        cols = rng.choice([_log(rng, 64, 8192), 128 * rng.randint(1, 64), 16 * rng.randint(4, 512)])
        return _quantize("", _log(rng, 1, 8192), cols, dtype, rng.random() < 0.4, layout)
    if kind == "matmul":
        tokens = _log(rng, 1, 8192)
        n = rng.choice([128 * rng.randint(1, 64), _log(rng, 64, 8192)])
        k = 16 * _log(rng, 16, 448)
        while tokens * n * k > 8192 * 4096 * 7168:
            n = max(64, n // 2)
        return _matmul("", tokens, n, k, dtype, layout)
    experts = rng.choice([8, 32, 64, 160, 256])
    local = rng.choice([experts, max(1, experts // 8)]) if kind == "combine" else experts
    hidden = rng.choice([8 * _log(rng, 32, 896), _log(rng, 256, 7168)])
    most = 8192 if dtype != "fp32" else 4096
    if kind == "train":
        most //= 2
    return _tokens("", kind, _log(rng, 1, most), hidden, rng.choice([1, 2, 4, 6, 8]), experts, local,
                   rng.randrange(experts - local + 1), rng.choice([1, 1, 16, 128]), dtype, rng.random() < 0.5)


def _rows(c):
    """Rows of the sorted tensors: every pair, and room to start each expert on a multiple of ``align``."""
    pairs, a = c["tokens"] * c["top_k"], c["align"]
    return -(-(pairs + (a - 1) * min(c["local"], pairs)) // a) * a


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed)
    c, T, dt = case, case["tokens"], DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if c["op"] == "quantize":
        width = c["cols"] * (2 if c["swiglu"] else 1)
        # activations: channels of unequal size, a few of them far out
        x = randn(T, width) * torch.exp(randn(width)).clamp_max(50.0)
        return dict(case=c, x=x.to(dt))
    if c["op"] == "matmul":
        x = randn(T, c["k"]) * torch.exp(0.5 * randn(c["k"]))
        a, sa = _plain_quantize(x, False, c["layout"])
        b, sb = _quantize_weight(randn(c["n"], c["k"]) * 0.02)
        return dict(case=c, a=a, sa=sa, b=b, sb=sb)
    # a router's choice: some experts are liked more than others, no expert twice for a token
    liked = randn(T, c["experts"]) + 0.5 * randn(c["experts"])
    top, ids = torch.topk(liked, c["top_k"], dim=1)
    ids = ids if c["wide"] else ids.int()
    weights = torch.softmax(top, dim=1)
    state = dict(case=c, ids=ids, weights=weights)
    rows, H = _rows(c), c["hidden"]
    if c["op"] in ("dispatch", "train"):
        state["x"] = randn(T, H).to(dt)
    if c["op"] in ("combine", "train"):
        state["y"] = randn(rows, H).to(dt)
    if c["op"] == "train":
        state["grads"] = (randn(rows, H).to(dt), randn(T, H).to(dt))
        for name in ("x", "y", "weights"):
            state[name].requires_grad_(True)
    return state


def run(state):
    c = state["case"]
    if own:
        return _run_own(c, state)
    if c["op"] == "quantize":
        return _plain_quantize(state["x"], c["swiglu"], c["layout"])
    if c["op"] == "matmul":
        return _plain_matmul(state["a"], state["sa"], state["b"], state["sb"], c["layout"], DTYPES[c["dtype"]])
    order = _plain_sort(state["ids"], c)
    if c["op"] == "dispatch":
        return dict(order, rows=_plain_permute(state["x"], order))
    if c["op"] == "combine":
        return _plain_unpermute(state["y"], order["pos"], state["weights"])
    with torch.no_grad():
        x, y, w = state["x"], state["y"], state["weights"]
        d_rows, d_out = state["grads"]
        return dict(rows=_plain_permute(x, order), out=_plain_unpermute(y, order["pos"], w),
                    dx=_plain_unpermute(d_rows, order["pos"], None), **_plain_unpermute_grads(d_out, y, order["pos"], w))


def _run_own(c, state):
    from fused_moe_b200 import ops
    if c["op"] == "quantize":
        return ops.quantize(state["x"], swiglu=c["swiglu"], scale_layout=c["layout"])
    if c["op"] == "matmul":
        return ops.block_matmul(state["a"], state["sa"], state["b"], state["sb"], scale_layout=c["layout"],
                                out_dtype=DTYPES[c["dtype"]])
    order = ops.sort_tokens(state["ids"], c["local"], c["offset"], align=c["align"])
    if c["op"] == "dispatch":
        return dict(offsets=order.offsets, pos=order.pos, pair=order.pair, rows=ops.permute(state["x"], order))
    if c["op"] == "combine":
        return ops.unpermute(state["y"], order, state["weights"])
    x, y, w = state["x"], state["y"], state["weights"]
    rows, out = ops.permute(x, order), ops.unpermute(y, order, w)
    dx, dy, dw = torch.autograd.grad((rows, out), (x, y, w), state["grads"])
    return dict(rows=rows, out=out, dx=dx, dy=dy, dw=dw)


# ---- the operators in elementary operations ----

def _blocks(x):
    """[T, K] -> [T, ceil(K/128), 128], zeros behind the last column."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).view(x.shape[0], -1, BLOCK)


def _plain_quantize(x, swiglu, layout):
    x = x.float()
    if swiglu:
        gate, up = x.chunk(2, dim=1)
        x = gate * (up * (1.0 / (1.0 + torch.exp(-up))))
    xb = _blocks(x)
    s = xb.abs().amax(-1).clamp_min(AMAX_MIN)
    s = s / torch.full_like(s, E4M3_MAX)   # (a division; by a plain number torch multiplies with its reciprocal)
    q = (xb / s[..., None]).view(x.shape[0], -1)[:, :x.shape[1]].contiguous().to(torch.float8_e4m3fn)
    return q, (s.t().contiguous() if layout == "kt" else s)


def _quantize_weight(w):
    n, k = w.shape
    wb = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK)).view(-(-n // BLOCK), BLOCK, -(-k // BLOCK), BLOCK)
    s = wb.abs().amax((1, 3)).clamp_min(AMAX_MIN) / E4M3_MAX
    q = (wb / s[:, None, :, None]).view(-(-n // BLOCK) * BLOCK, -1)[:n, :k].contiguous().to(torch.float8_e4m3fn)
    return q, s


def _plain_matmul(a, sa, b, sb, layout, dtype):
    n, k = b.shape
    sa = sa.t() if layout == "kt" else sa
    a = a.float() * sa.repeat_interleave(BLOCK, 1)[:, :k]
    b = b.float() * sb.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return torch.matmul(a, b.t()).to(dtype)


def _plain_sort(ids, c):
    dev, pairs, rows = ids.device, ids.numel(), _rows(c)
    e = ids.reshape(-1).long() - c["offset"]
    e = torch.where((e >= 0) & (e < c["local"]), e, c["local"])
    sorted_e, pair_of = torch.sort(e, stable=True)
    counts = torch.bincount(e, minlength=c["local"] + 1)
    first = torch.cumsum(counts, 0) - counts                      # in the list of pairs
    padded = -(-counts[:-1] // c["align"]) * c["align"]
    offsets = torch.nn.functional.pad(torch.cumsum(padded, 0), (1, 0))
    row = offsets[sorted_e] + torch.arange(pairs, device=dev) - first[sorted_e]
    row = torch.where(sorted_e < c["local"], row, -1)
    pos = torch.empty(pairs, dtype=torch.int32, device=dev)
    pos[pair_of] = row.int()
    pair = torch.full((rows + 1,), -1, dtype=torch.int32, device=dev)
    pair[row] = pair_of.int()                                     # (row -1: the extra element)
    return dict(offsets=offsets.int(), pos=pos.view(ids.shape), pair=pair[:-1])


def _plain_permute(x, order):
    top_k = order["pos"].shape[1]
    kept = (order["pair"] >= 0)[:, None]
    return torch.where(kept, x[order["pair"].clamp_min(0).long() // top_k], torch.zeros((), dtype=x.dtype, device=x.device))


def _plain_unpermute(y, pos, weights):
    kept = (pos >= 0)[..., None]
    v = torch.where(kept, y[pos.clamp_min(0).long()].float(), 0.0)
    if weights is not None:
        v = v * weights[..., None]
    return v.sum(1).to(y.dtype)


def _plain_unpermute_grads(d_out, y, pos, weights):
    kept, d = (pos >= 0)[..., None], d_out.float()[:, None, :]
    at = pos.clamp_min(0).long()
    dw = torch.where(kept, d * y[at].float(), 0.0).sum(-1)
    dy = torch.zeros((y.shape[0] + 1, y.shape[1]), dtype=y.dtype, device=y.device)
    dy[pos.long().reshape(-1)] = (d * weights[..., None]).to(y.dtype).reshape(-1, y.shape[1])
    return dict(dy=dy[:-1], dw=dw)


# ---- the same from the definitions in 64 bits ----

def _e4m3(v):
    """Nearest e4m3 value (ties to even) of float64 ``v``, at most 448 in size: steps of 2^(e-3), none below 2^-9."""
    step = torch.exp2((torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -30)))).clamp_min(-6.0) - 3.0)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def exact(case, seed):
    c = case
    s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    if c["op"] == "quantize":
        x = s["x"].double()
        if c["swiglu"]:
            x = x[:, :c["cols"]] * x[:, c["cols"]:] * torch.sigmoid(x[:, c["cols"]:])
        codes, scales = [], []
        for k0 in range(0, c["cols"], BLOCK):
            xb = x[:, k0:k0 + BLOCK]
            # the scale is a number of 32 bits, and so is the quotient that is rounded to a code
            sb = (xb.abs().amax(1).float().clamp_min(AMAX_MIN).double() / E4M3_MAX).float().double()
            codes.append(_e4m3((xb / sb[:, None]).float().double()))
            scales.append(sb)
        return torch.cat(codes, 1), torch.stack(scales, 0 if c["layout"] == "kt" else 1)
    if c["op"] == "matmul":
        k = torch.arange(c["k"], device=s["a"].device) // BLOCK
        n = torch.arange(c["n"], device=s["a"].device) // BLOCK
        sa = s["sa"].double() if c["layout"] == "tk" else s["sa"].double().t()
        a = s["a"].double() * sa[:, k]
        b = s["b"].double() * s["sb"].double()[n][:, k]
        return torch.einsum("mk,nk->mn", a, b)
    # rows by counting: how many pairs of the same expert come before, behind the padded segments of the experts before
    ids, T, K, H = s["ids"].long().reshape(-1) - c["offset"], c["tokens"], c["top_k"], c["hidden"]
    local = (ids >= 0) & (ids < c["local"])
    row = torch.zeros_like(ids)
    start = 0
    for e in range(c["local"]):
        mine = ids == e
        n = torch.cumsum(mine.long(), 0)
        row += torch.where(mine, start + n - 1, 0)
        start += -(-int(n[-1]) // c["align"]) * c["align"]
    at, pair = row[local], torch.nonzero(local).squeeze(1)
    rows = _rows(c)

    def scatter(values):
        out = torch.zeros(rows, H, dtype=torch.float64, device=ids.device)
        out[at] = values
        return out

    def gather(values, w):
        v = values.double()[at]
        v = v if w is None else v * w.double().reshape(-1)[pair][:, None]
        return torch.zeros(T, H, dtype=torch.float64, device=ids.device).index_add_(0, pair // K, v)

    if c["op"] == "dispatch":
        return dict(offsets=None, pos=None, pair=None, rows=scatter(s["x"].double()[pair // K]))
    if c["op"] == "combine":
        return gather(s["y"], s["weights"])
    d_rows, d_out = s["grads"]
    dw = torch.zeros(T * K, dtype=torch.float64, device=ids.device)
    dw[pair] = (d_out.double()[pair // K] * s["y"].double()[at]).sum(1)
    return dict(rows=scatter(s["x"].double()[pair // K]), out=gather(s["y"], s["weights"]), dx=gather(d_rows, None),
                dy=scatter(d_out.double()[pair // K] * s["weights"].double().reshape(-1)[pair][:, None]),
                dw=dw.view(T, K))


def work(case):
    c, T = case, case["tokens"]
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "quantize":
        n = T * c["cols"]
        return {"bytes": n * size * (2 if c["swiglu"] else 1) + n + 4 * T * -(-c["cols"] // BLOCK), "flops": 4 * n}
    if c["op"] == "matmul":
        n, k = c["n"], c["k"]
        blocks = -(-k // BLOCK)
        return {"bytes": (T + n) * k + 4 * blocks * (T + -(-n // BLOCK)) + T * n * size, "flops": 2 * T * n * k}
    pairs, H, rows = T * c["top_k"], c["hidden"], _rows(c)
    held = pairs * c["local"] // c["experts"]                       # pairs of a local expert, if the router is fair
    sort = pairs * (8 if c["wide"] else 4)
    if c["op"] == "dispatch":
        return {"bytes": sort + 4 * (pairs + rows + c["local"] + 1) + (T + rows) * H * size, "flops": pairs}
    if c["op"] == "combine":
        return {"bytes": sort + 4 * pairs + (held + T) * H * size, "flops": 2 * held * H}
    # permute, unpermute; dx; dy and dw
    return {"bytes": sort + 12 * pairs + ((T + rows) + (held + T) + (held + T) + (T + held + rows)) * H * size,
            "flops": 7 * held * H}
