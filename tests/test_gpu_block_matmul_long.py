"""A product that keeps one launch busy for longer than any single wait in it may last: the bounded waits are each of a hand-off's
length, so nothing gives up and nothing is reported."""
import pytest
import torch

from fused_moe_b200 import _capi

pytestmark = pytest.mark.gpu
WAIT_BUDGET_CYCLES = 400_000_000                 # of a bounded device-side wait (csrc/common.cuh)


def test_a_launch_longer_than_the_budget_of_a_wait():
    """Codes of 0 and 1, scales of one: every partial sum is a whole number below 2^24, so rows are exact in fp32; the result is
    rounded once to bf16."""
    dev = torch.device("cuda", 0)
    n = 81920                                    # 1.1e15 operations; operands of 6.7 GB each, a result of 13.4 GB
    if torch.cuda.mem_get_info(dev)[0] < 36 << 30:
        pytest.skip("needs 36 GB of device memory")
    one, kb = 0x38, n // 128
    g = torch.Generator(device=dev).manual_seed(0)
    a = torch.randint(0, 2, (n, n), generator=g, device=dev, dtype=torch.uint8).mul_(one)
    b = torch.randint(0, 2, (n, n), generator=g, device=dev, dtype=torch.uint8).mul_(one)
    sa, sb = torch.ones(kb, n, device=dev), torch.ones(kb, kb, device=dev)
    out = torch.empty(n, n, device=dev, dtype=torch.bfloat16)
    status = torch.zeros(4, dtype=torch.int32).pin_memory()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    stream = torch.cuda.current_stream(dev)
    begin.record()
    rc = _capi.lib().b200moe_block_matmul(a.data_ptr(), n, sa.data_ptr(), 1, n, b.data_ptr(), n, sb.data_ptr(), kb, 1, n, n, n,
                                          out.data_ptr(), _capi.BF16, n, status.data_ptr(), stream.cuda_stream)
    end.record()
    torch.cuda.synchronize()
    assert rc == 0
    # (at the highest clock there is, 1965 MHz, the launch has to take longer than the budget to test anything)
    assert begin.elapsed_time(end) * 1e-3 * 1.965e9 > 2 * WAIT_BUDGET_CYCLES
    assert status.tolist() == [0, 0, 0, 0]
    at = [0, 1, 127, 128, 255, 256, n // 2, n // 2 + 77, n - 257, n - 129, n - 128, n - 1]
    want = ((a[at] != 0).float() @ (b[:4096] != 0).float().t(), (a[at] != 0).float() @ (b[-4096:] != 0).float().t())
    assert torch.equal(out[at, :4096], want[0].bfloat16()) and torch.equal(out[at, -4096:], want[1].bfloat16())
