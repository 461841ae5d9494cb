"""``block_matmul`` against the formula in 64 bits: exactly where every sum is representable in fp32, else within the bound of
fp32 summation in any order."""
import pytest
import torch

import fused_moe_b200 as F
from fused_moe_b200 import MoEError, synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}

SHAPES = [(1, 1, 16), (1, 128, 128), (2, 130, 144), (7, 64, 272), (8, 4096, 7168), (9, 1000, 1024), (16, 512, 2048), (17, 129, 400),
          (33, 257, 1168), (64, 7168, 2048), (65, 300, 640), (127, 384, 4096), (128, 128, 128), (129, 513, 256), (200, 1001, 7168),
          (256, 576, 1536), (300, 2048, 512), (511, 255, 2064), (1025, 1152, 896), (2048, 2304, 1024), (4100, 520, 384),
          (129, 7168, 16384), (4200, 4224, 400), (2500, 5000, 1936)]


def expand(sa, sb, N, K):
    """Scales per element: [M, K] and [N, K], fp64."""
    return (sa.double().repeat_interleave(128, 1)[:, :K],
            sb.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K])


def small_whole_numbers(M, N, K, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randint(-4, 5, s, generator=g, device=DEV).float()           # noqa: E731
    p = lambda *s: torch.exp2(torch.randint(-1, 2, s, generator=g, device=DEV).float())   # noqa: E731
    kb = -(-K // 128)
    return (r(M, K).to(torch.float8_e4m3fn), p(M, kb) * torch.where(torch.arange(M, device=DEV) % 3 == 0, -1.0, 1.0)[:, None],
            r(N, K).to(torch.float8_e4m3fn), p(-(-N // 128), kb))


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("layout", ["tk", "kt"])
def test_exact_where_fp32_is(M, N, K, layout):
    """Codes of at most 4 and scales 1/2, 1, 2 (some negative): every partial sum is a multiple of 1/4 below 2^20."""
    a, sa, b, sb = small_whole_numbers(M, N, K, M + N + K)
    ea, eb = expand(sa, sb, N, K)
    ref = (a.double() * ea) @ (b.double() * eb).t()
    out = F.block_matmul(a, sa.t().contiguous() if layout == "kt" else sa, b, sb, scale_layout=layout, out_dtype=torch.float32)
    assert torch.equal(out.double(), ref)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 4096, 7168), (5, 1000, 528), (24, 2048, 2048), (100, 640, 7168), (301, 1001, 1024), (1500, 768, 2304)])
def test_real_data_within_the_bound_of_fp32_sums(M, N, K, dtype):
    """At most 128 + K/128 additions, each off by at most one ulp (2^-23: tensor cores may truncate), of terms whose absolute
    values sum to S: |error| <= (128 + K/128 + 2) 2^-23 S, then half an ulp of the result's type."""
    g = torch.Generator(device=DEV).manual_seed(M)
    a, sa = F.quantize(torch.randn(M, K, generator=g, device=DEV) * torch.exp(torch.randn(K, generator=g, device=DEV)))
    w = 0.02 * torch.randn(-(-N // 128) * 128, -(-K // 128) * 128, generator=g, device=DEV)
    b, sb = synth.quant_blocks_128x128(w)
    b = b[:N, :K].contiguous()
    out = F.block_matmul(a, sa, b, sb, out_dtype=dtype)
    ea, eb = expand(sa.t(), sb, N, K)
    x, y = a.double() * ea, b.double() * eb
    ref, mass = x @ y.t(), x.abs() @ y.abs().t()
    bound = (130 + -(-K // 128)) * 2.0 ** -23 * mass
    bound = bound + HALF_ULP[dtype] * (ref.abs() + bound) + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert ((out.double() - ref).abs() <= bound).all()
    assert torch.equal(out, F.block_matmul(a, sa, b, sb, out_dtype=dtype)), "results repeat bit for bit"


def test_strides_of_everything():
    M, N, K = 70, 200, 400
    a, sa, b, sb = small_whole_numbers(M, N, K, 1)
    ea, eb = expand(sa, sb, N, K)
    ref = (a.double() * ea) @ (b.double() * eb).t()
    wide_a = torch.zeros(M, K + 48, dtype=torch.uint8, device=DEV)
    wide_a[:, 16:16 + K] = a.view(torch.uint8)
    wide_b = torch.zeros(N, K + 32, dtype=torch.uint8, device=DEV)
    wide_b[:, 32:] = b.view(torch.uint8)
    odd_a = torch.zeros(M, K + 5, dtype=torch.uint8, device=DEV)       # neither pitch nor start on 16 bytes: copied
    odd_a[:, 3:3 + K] = a.view(torch.uint8)
    far = torch.zeros(M, 3 * sa.shape[1], device=DEV)
    far[:, ::3] = sa
    sbt = sb.t().contiguous().t()
    for av in (wide_a[:, 16:16 + K], odd_a[:, 3:3 + K], a.t().contiguous().t()):
        for start in (0, 1):
            host = torch.full((M, N + 9), 7.0, device=DEV)
            out = F.block_matmul(av, far[:, ::3], wide_b[:, 32:], sbt, scale_layout="tk", out=host[:, start:start + N])
            assert out.data_ptr() == host[:, start:].data_ptr()
            assert torch.equal(out.double(), ref)
            assert (host[:, :start] == 7).all() and (host[:, start + N:] == 7).all(), "columns beside the result stay"
    for dt in (torch.bfloat16, torch.float16):
        host = torch.full((M, N + 3), 7.0, device=DEV, dtype=dt)
        F.block_matmul(a, sa, b, sb, scale_layout="tk", out=host[:, 1:1 + N])
        assert torch.equal(host[:, 1:1 + N], ref.to(dt)) and (host[:, 0] == 7).all() and (host[:, 1 + N:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(300, 77, 128), (130, 256, 64), (70, 200, 2048), (3000, 1, 128), (4200, 1301, 256), (2600, 2176, 400)])
def test_result_rows_that_start_anywhere(M, N, K, dtype):
    """Rows of the result on every boundary of their elements, by start and by pitch; what lies beside them stays."""
    a, sa, b, sb = small_whole_numbers(M, N, K, 2)
    ea, eb = expand(sa, sb, N, K)
    ref = ((a.double() * ea) @ (b.double() * eb).t()).to(dtype)
    for start, pitch in [(s, N + 17 + s % 2) for s in range(17)] + [(s, -(-(N + 16) // 32) * 32) for s in (0, 1, 4, 8, 15, 16)]:
        host = torch.full((M + 2, pitch), 7.0, device=DEV, dtype=dtype)
        F.block_matmul(a, sa, b, sb, scale_layout="tk", out=host[1:-1, start:start + N])
        assert torch.equal(host[1:-1, start:start + N], ref), (start, pitch)
        host[1:-1, start:start + N] = 7.0
        assert (host == 7).all(), (start, pitch)


@pytest.mark.parametrize("M", [3, 40, 200, 700])
def test_not_a_number_stays_in_its_row_and_column(M):
    N, K = 300, 1024
    a, sa, b, sb = small_whole_numbers(M, N, K, 9)
    ea, eb = expand(sa, sb, N, K)
    ref = (a.double() * ea) @ (b.double() * eb).t()
    a, b, sa = a.view(torch.uint8).clone(), b.view(torch.uint8).clone(), sa.clone()
    a[1, 700] = 0x7f
    b[255, 3] = 0xff
    sa[2, 7] = float("inf")
    out = F.block_matmul(a, sa, b, sb, scale_layout="tk", out_dtype=torch.float32)
    bad = torch.zeros(M, N, dtype=torch.bool, device=DEV)
    bad[1], bad[2], bad[:, 255] = True, True, True
    assert out[1].isnan().all() and out[:, 255].isnan().all() and not out[2].isfinite().any()
    assert torch.equal(torch.where(bad, 0.0, out.double()), torch.where(bad, 0.0, ref))


def test_empty_extents_and_refusals():
    a, sa, b, sb = small_whole_numbers(4, 8, 256, 3)
    assert F.block_matmul(a[:0], sa[:0], b, sb, scale_layout="tk").shape == (0, 8)
    assert F.block_matmul(a, sa, b[:0], sb[:0], scale_layout="tk").shape == (4, 0)
    ok = dict(scale_layout="tk")
    with pytest.raises(TypeError):
        F.block_matmul(a.float(), sa, b, sb, **ok)
    with pytest.raises(TypeError):
        F.block_matmul(a, sa.double(), b, sb, **ok)
    with pytest.raises(TypeError):
        F.block_matmul(a, sa, b, sb, out_dtype=torch.float64, **ok)
    with pytest.raises(ValueError):
        F.block_matmul(a, sa, b, sb)                                 # scales are not [K/128, M]
    with pytest.raises(ValueError):
        F.block_matmul(a, sa, b[:, :128], sb, **ok)
    with pytest.raises(ValueError):
        F.block_matmul(a[:, :200].contiguous(), sa, b[:, :200].contiguous(), sb, **ok)
    with pytest.raises(ValueError):
        F.block_matmul(a, sa, b.t().contiguous().t(), sb, **ok)
    for rows in (1, 4):                                                 # elements apart, in one row and in several
        with pytest.raises(ValueError):
            F.block_matmul(a, sa, torch.zeros(rows, 2 * a.shape[1], dtype=torch.uint8, device=DEV)[:, ::2], sb[:1], **ok)
    with pytest.raises(ValueError):                                     # rows that overlap in steps of a row
        F.block_matmul(a, sa, torch.zeros(4 * a.shape[1], dtype=torch.uint8, device=DEV).as_strided((3, a.shape[1]), (a.shape[1], 2)), sb[:1], **ok)
    with pytest.raises(ValueError):
        F.block_matmul(a, sa, b, sb[:, :1], **ok)
    with pytest.raises(ValueError):
        F.block_matmul(a, sa, b, sb, out=torch.zeros(4, 9, device=DEV), **ok)
    with pytest.raises(ValueError):
        F.block_matmul(a, sa, b, sb, out=torch.zeros(8, 4, device=DEV).t(), **ok)
    with pytest.raises(RuntimeError):
        F.block_matmul(a, sa, b, sb.cpu(), **ok)
    with pytest.raises(RuntimeError, match="no gradient"):
        F.block_matmul(a, sa.clone().requires_grad_(True), b, sb, **ok)
    with pytest.raises(RuntimeError, match="no gradient"):
        F.block_matmul(a, sa, b.clone().view(torch.float8_e4m3fn).requires_grad_(True), sb, **ok)
    assert issubclass(MoEError, RuntimeError)
