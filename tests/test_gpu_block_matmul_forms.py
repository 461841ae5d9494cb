"""``block_matmul`` in every form that its rule of sizes can choose: which shapes take which form is asserted on the host, each
form's results are exact where fp32 is, in every type of result."""
import pytest
import torch

import fused_moe_b200 as F
from fused_moe_b200 import _capi
from test_gpu_block_matmul import DEV, expand, small_whole_numbers

SMS = 148
# form (0: CTA pairs; S: parts of K, CTAs alone on their SMs; 16 + S: two on an SM) -> shapes: one row, odd and even widths, rows
# of a last tile that is not full
FORMS = {
    0: [(600, 7553, 16), (2138, 4608, 704), (3709, 4481, 1264), (8000, 1536, 2080)],
    1: [(1, 64, 16), (2, 65, 128), (134, 67, 144), (300, 1024, 240)],
    2: [(1, 64, 400), (5, 71, 416), (131, 2689, 1744), (140, 2816, 1808)],
    3: [(1, 65, 656), (12, 2505, 1152), (37, 2512, 1152), (133, 2301, 1488), (4175, 64, 1712)],
    4: [(1, 64, 944), (3, 69, 960), (130, 77, 1520), (160, 96, 1760)],
    8: [(1, 65, 2000), (30, 67, 2032), (132, 71, 2704), (160, 96, 2720)],
    17: [(263, 6361, 16), (260, 6352, 144), (1300, 1701, 128)],
    18: [(135, 5597, 8928), (5885, 144, 8640)],
    19: [(245, 5371, 12992), (129, 4797, 4112), (5407, 144, 3872)],
    20: [(62, 6591, 16224), (134, 4271, 3424), (147, 4432, 3440)],
    24: [(1, 4144, 3840), (3, 4235, 4800), (10, 4293, 4800)],
}
SHAPES = [s for shapes in FORMS.values() for s in shapes]


def form(M, N, K, pitch=None):
    return _capi.lib().b200moe_block_matmul_form(M, N, K, pitch or K, K, SMS)


def test_the_shapes_below_take_every_form():
    for want, shapes in FORMS.items():
        for s in shapes:
            assert form(*s) == want, s
    # and there are no others: every kind of size, coarsely
    seen = set()
    for M in (1, 2, 3, 9, 20, 70, 128, 134, 147, 245, 300, 600, 1300, 2500, 5500, 8192):
        for N in (1, 64, 144, 640, 1411, 2512, 4144, 4432, 5371, 6352, 8192):
            for K in (16, 128, 144, 400, 656, 944, 1152, 2000, 3440, 4800, 8640, 12992, 16224):
                seen.add(form(M, N, K))
    assert seen <= set(FORMS)


def test_refusals_of_the_question():
    f = _capi.lib().b200moe_block_matmul_form
    assert f(0, 8, 128, 128, 128, SMS) == -1 and f(8, 0, 128, 128, 128, SMS) == -1 and f(8, 8, 0, 128, 128, SMS) == -1
    assert f(8, 8, 128, 112, 128, SMS) == -1 and f(8, 8, 128, 128, 112, SMS) == -1 and f(8, 8, 128, 128, 128, 0) == -1
    assert f(8, 8, 120, 128, 128, SMS) == -2 and f(0x7fffffff, 8, 128, 128, 128, SMS) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_exact_in_every_form_and_type(M, N, K):
    """Codes of at most 4 and scales 1/2, 1, 2 (some negative): every partial sum is a multiple of 1/4 below 2^20, so the sum is
    exact in fp32 in any order and the result is its one rounding."""
    if torch.cuda.get_device_properties(0).multi_processor_count != SMS:
        pytest.skip("the forms are those of 148 SMs")
    a, sa, b, sb = small_whole_numbers(M, N, K, M + N + K)
    ea, eb = expand(sa, sb, N, K)
    ref = ((a.double() * ea) @ (b.double() * eb).t()).float()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        out = torch.full((M, N + 6), 7.0, dtype=dtype, device=DEV)
        F.block_matmul(a, sa, b, sb, scale_layout="tk", out=out[:, 3:N + 3])     # rows that start off 16 bytes, guards beside them
        assert torch.equal(out[:, 3:N + 3], ref.to(dtype)), dtype
        assert (out[:, :3] == 7).all() and (out[:, N + 3:] == 7).all()
        assert torch.equal(F.block_matmul(a, sa.t().contiguous(), b, sb, out_dtype=dtype), ref.to(dtype)), dtype
