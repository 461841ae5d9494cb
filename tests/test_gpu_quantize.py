"""``quantize``: codes and scales are integers of an exact formula, so they are compared bit for bit with the formula in torch on
the CPU (fp32 division is correctly rounded there); behind a SwiGLU, whose exponential is not exactly rounded, with 64 bits."""
import pytest
import torch

import fused_moe_b200 as F
from fused_moe_b200 import synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def formula(x):
    """fp32 [T, K] on the CPU -> (codes as uint8 [T, K], scales [T, blocks])."""
    T, K = x.shape
    xb = torch.nn.functional.pad(x.float(), (0, -K % 128)).view(T, -(-K // 128), 128)
    m = xb.abs().amax(-1)
    s = torch.where(m < 1e-12, torch.tensor(1e-12), m) / torch.full_like(m, 448.0)
    q = (xb / s[..., None]).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).view(T, -(-K // 128) * 128)[:, :K], s


def check(x, x_cpu=None, **kw):
    q, s = F.quantize(x, **kw)
    qr, sr = formula((x.cpu() if x_cpu is None else x_cpu))
    s = s.cpu().t() if kw.get("scale_layout", "kt") == "kt" else s.cpu()
    assert torch.equal(s, sr) or torch.equal(torch.nan_to_num(s, 7.0), torch.nan_to_num(sr, 7.0))
    q = q.view(torch.uint8).cpu()
    nan = lambda c: (c & 0x7f) == 0x7f                                     # noqa: E731  (the sign of a NaN is free)
    assert torch.equal(nan(q), nan(qr))
    assert torch.equal(torch.where(nan(q), 0, q), torch.where(nan(qr), 0, qr))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7168), (3, 128), (63, 129), (64, 256), (65, 127), (200, 1000), (130, 8), (35, 1100), (300, 600), (17, 2048)])
@pytest.mark.parametrize("layout", ["kt", "tk"])
def test_codes_and_scales_are_the_formulas(dtype, rows, cols, layout):
    g = torch.Generator().manual_seed(rows * 1000 + cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(cols, generator=g))).to(dtype)
    check(x.to(DEV), x, scale_layout=layout)


def test_same_bits_as_the_synthetic_inputs():
    x = torch.randn(37, 1024, generator=torch.Generator().manual_seed(5))
    q, s = F.quantize(x.to(DEV))
    qr, sr = synth.quant_rows_1x128(x)
    assert torch.equal(q.view(torch.uint8).cpu(), qr.view(torch.uint8)) and torch.equal(s.cpu(), sr)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_unaligned_rows(dtype):
    big = torch.randn(70, 700, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    check(big[:, 8:520])                # aligned start, padded rows
    check(big[:, 3:400])                # neither
    check(big[::2, 5:300])
    check(big.t()[100:300])             # inner stride: copied
    check(big[:1, 1:2])
    check(torch.empty(0, 256, dtype=dtype, device=DEV), torch.empty(0, 256))


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 7), (torch.float16, 10)])
def test_every_quotient_of_a_16_bit_type(dtype, bits):
    """Every mantissa of the block's maximum against every smaller value of eleven binades: all quotients that can lie next to a
    border of two codes (a quotient's bits depend on the two mantissas and the difference of the exponents)."""
    one = 1 << bits
    vals = (torch.arange(one, dtype=torch.float64) / one + 1.0)
    small = torch.cat([vals * 2.0 ** -e for e in range(0, 12)])
    small = small[torch.randperm(len(small), generator=torch.Generator().manual_seed(1))]
    small = torch.cat([small, torch.zeros(-len(small) % 127, dtype=torch.float64)]).view(-1, 127)
    sign = torch.where(torch.arange(127) % 2 == 0, 1.0, -1.0)
    step = max(1, one // 128)           # 128 maxima at a time
    for m0 in range(0, one, 128 * step if dtype == torch.float16 else one):
        amax = vals[m0:m0 + 128 * step][::1 if dtype == torch.bfloat16 else 8]
        x = torch.cat([amax[:, None, None].expand(-1, small.shape[0], 1), torch.minimum(small[None], amax[:, None, None]) * sign], 2)
        x = x.reshape(-1, 128).to(dtype).to(DEV)
        q, s = F.quantize(x)
        f = x.float()
        sr = f.abs().amax(1) / torch.full((len(f),), 448.0, device=DEV)      # tensor / tensor: a correctly rounded division
        assert torch.equal(s[0], sr)
        assert torch.equal(q.view(torch.uint8), (f / sr[:, None]).to(torch.float8_e4m3fn).view(torch.uint8))


def test_fp32_quotients_next_to_borders():
    """x = RN(s * border) and its neighbours, for scales of every kind: the quotient lies within an ulp of a tie of two codes."""
    g = torch.Generator().manual_seed(3)
    amax = torch.exp(8 * torch.randn(4096, generator=g)).float()
    s = amax / torch.full_like(amax, 448.0)
    codes = torch.arange(0, 126, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    ties = ((codes[1:] + codes[:-1]) / 2)[torch.randint(0, 125, (4096, 42), generator=g)]
    near = (ties * s.double()[:, None]).float()
    x = torch.cat([near, torch.nextafter(near, torch.tensor(0.0)), torch.nextafter(near, torch.tensor(1e38)),
                   torch.zeros(4096, 1), amax[:, None]], 1)
    assert x.shape[1] == 128
    check(x.to(DEV), x)


@pytest.mark.parametrize("dtype", TYPES)
def test_special_values(dtype):
    inf, nan = float("inf"), float("nan")
    x = torch.randn(12, 256, generator=torch.Generator().manual_seed(4)).to(dtype)
    x[0] = 0.0
    x[1, :128] = -0.0
    x[2, 5] = inf
    x[3, 200] = -inf
    x[4, 0] = nan
    x[5, 7], x[5, 9] = nan, inf
    x[6] = torch.finfo(dtype).max
    x[7] = torch.finfo(dtype).tiny
    x[8] = torch.finfo(dtype).smallest_normal / 4
    x[9, ::2] = 1e-13
    x[10, :128] = inf
    x[11] = -torch.finfo(dtype).max
    check(x.to(DEV), x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 2048), (67, 128), (5, 130), (33, 1), (64, 264)])
def test_swiglu_form(dtype, rows, cols):
    """|code * scale - x| is half a step of e4m3 (2^-4 of the value, 2^-10 scales below its normal range) plus what fp32 makes of
    the SwiGLU: an exponential and a reciprocal within an ulp (2^-23 each), three roundings of half an ulp, below 2^-21 together."""
    g = torch.Generator().manual_seed(rows + cols)
    x = (4 * torch.randn(rows, 2 * cols, generator=g)).to(dtype)
    q, s = F.quantize(x.to(DEV), swiglu=True, scale_layout="tk")
    d = x.double()
    ref = d[:, :cols] * d[:, cols:] * torch.sigmoid(d[:, cols:])
    blocks = torch.nn.functional.pad(ref, (0, -cols % 128)).view(rows, -1, 128).abs().amax(-1)
    sr = blocks.clamp_min(1e-12) / 448
    assert ((s.cpu().double() - sr).abs() <= sr * (2.0 ** -21 + 2.0 ** -23)).all()
    se = s.cpu().double().repeat_interleave(128, 1)[:, :cols]
    err = (q.float().cpu().double() * se - ref).abs()
    assert (err <= torch.maximum(2.0 ** -4 * ref.abs(), 2.0 ** -10 * se) * (1 + 2.0 ** -20) + 2.0 ** -21 * ref.abs()).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_swiglu_special_values(dtype):
    """Infinities, NaN and zeros go through g * (u * (1 / (1 + exp(-u)))) and the block as the formula says, from fp32 on."""
    inf, nan = float("inf"), float("nan")
    pairs = [(0.0, 0.0), (-0.0, 3.0), (1.0, inf), (1.0, -inf), (inf, 1.0), (-inf, 2.0), (0.0, inf), (nan, 1.0), (1.0, nan),
             (2.0, -60000.0), (60000.0, 60000.0), (-60000.0, -3.0), (1.0, 100.0), (1.0, -100.0), (1e-7, 1e-7)]
    x = torch.ones(len(pairs), 2 * 256, dtype=torch.float32)
    for i, (g, u) in enumerate(pairs):
        x[i, 5], x[i, 256 + 5] = g, u
    x = x.to(dtype)
    q, s = F.quantize(x.to(DEV), swiglu=True, scale_layout="tk")
    f = x.float()
    f = f[:, :256] * (f[:, 256:] * (1.0 / (1.0 + torch.exp(-f[:, 256:]))))
    qr, sr = formula(f)
    fin = sr.isfinite()
    assert torch.equal(s.cpu()[~fin].nan_to_num(7.0), sr[~fin].nan_to_num(7.0))
    assert ((s.cpu()[fin] - sr[fin]).abs() <= 2.0 ** -20 * sr[fin]).all()
    qd, qrd = q.float().cpu(), qr.view(torch.float8_e4m3fn).float()
    assert torch.equal(qd.isnan(), qrd.isnan())
    # a quotient may take the neighbouring code: a step of e4m3 is at most 2^-3 of the value, 2^-9 below the normal range
    assert ((qd - qrd).nan_to_num(0.0).abs() <= torch.maximum(2.0 ** -3 * qrd.abs().nan_to_num(0.0), torch.tensor(2.0 ** -9))).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_swiglu_far_down(dtype):
    """1 + exp(-u) up to where the exponential overflows, whose reciprocal is below fp32's normal range, times large numbers: the
    scale within 2^-21 of the formula's (see test_swiglu_form) and half an ulp, 2^-24, of the division."""
    u = torch.tensor([-86.5, -87.0, -87.5, -88.0, -88.5, -40.0, -3.0]).to(dtype)
    x = torch.zeros(len(u), 256)
    x[:, 7], x[:, 128 + 7] = 1e37, u.float()
    x = x.to(dtype)
    q, s = F.quantize(x.to(DEV), swiglu=True, scale_layout="tk")
    d = x.double()
    ref = (d[:, 7] * d[:, 128 + 7] * torch.sigmoid(d[:, 128 + 7])).abs() / 448
    assert ((s.cpu()[:, 0].double() - ref).abs() <= ref * (2.0 ** -21 + 2.0 ** -23)).all()
    assert (q.float().cpu()[:, 7] == -448).all()


def test_refusals():
    x = torch.zeros(4, 256, device=DEV)
    with pytest.raises(TypeError):
        F.quantize(x.double())
    with pytest.raises(ValueError):
        F.quantize(x[0])
    with pytest.raises(ValueError):
        F.quantize(x, scale_layout="nk")
    with pytest.raises(ValueError):
        F.quantize(x[:, :255], swiglu=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        F.quantize(x.clone().requires_grad_(True))
