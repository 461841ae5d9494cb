"""``quantize`` of fp16 with every mantissa that a block's maximum can have, odd ones among them."""
import pytest
import torch

import fused_moe_b200 as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ONE = 1024                                       # mantissas of a binade


@pytest.mark.parametrize("first", range(0, ONE, 128))
def test_every_quotient_of_fp16(first):
    """Maxima of one binade, each against every value of the twenty binades from its own downwards that is not larger: down to
    where the codes end (448 against half of 2^-9 is 2^19).  A quotient's bits depend on the two mantissas alone, whether it
    lies next to a border of two codes on the difference of the exponents too."""
    vals = torch.arange(ONE, dtype=torch.float64) / ONE + 1.0
    small = torch.cat([vals * 2.0 ** (6 - e) for e in range(20)])
    small = small[torch.randperm(len(small), generator=torch.Generator().manual_seed(first))]
    small = torch.cat([small, torch.zeros(-len(small) % 127, dtype=torch.float64)]).view(-1, 127)
    sign = torch.where(torch.arange(127) % 2 == 0, 1.0, -1.0)
    amax = 64 * vals[first:first + 128]
    assert len(amax) == 128 and (amax / 64 * ONE).long().tolist() == list(range(ONE + first, ONE + first + 128))
    x = torch.cat([amax[:, None, None].expand(-1, small.shape[0], 1), torch.minimum(small[None], amax[:, None, None]) * sign], 2)
    x = x.reshape(-1, 128)
    assert torch.equal(x.half().double(), x)
    f = x.float().to(DEV)
    q, s = F.quantize(x.half().to(DEV))
    want = f.abs().amax(1) / torch.full((len(f),), 448.0, device=DEV)        # tensor / tensor: a correctly rounded division
    assert torch.equal(s[0], want)
    assert torch.equal(q.view(torch.uint8), (f / want[:, None]).to(torch.float8_e4m3fn).view(torch.uint8))
