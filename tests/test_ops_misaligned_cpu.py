"""Tables of 4-byte numbers that start off a multiple of four are refused by the C entry points, before any CUDA call."""
import ctypes as C

import pytest

from fused_moe_b200 import _capi

MISALIGNED = -6
BUFFER = C.create_string_buffer(1 << 16)
P = (C.addressof(BUFFER) + 255) // 256 * 256

# valid arguments of each call, and which of them are such tables
CALLS = {
    "b200moe_block_matmul": ([P, 256, P, 1, 4, P, 256, P, 2, 1, 4, 8, 256, P, 1, 8, P, None], (2, 7, 16)),
    "b200moe_quantize": ([P, 1, 256, 4, 256, 0, P, 256, P, 1, 4, None], (8,)),
    "b200moe_sort_tokens": ([P, 32, 8, 4, 8, 16, 0, 1, P, P, P, P, 32, None, 0, None], (0, 8, 9, 10, 11)),
    "b200moe_permute_rows": ([P, 512, 512, 2, 4, 8, P, P, P, 16, 32, P, 512, 1, None], (6, 7, 8)),
    "b200moe_unpermute_rows": ([P, 1, 256, P, P, 8, 4, 8, 256, P, 256, None], (3, 4)),
    "b200moe_unpermute_grad": ([P, 1, 256, P, 256, P, 8, P, P, P, 16, 4, 8, 256, 32, P, 256, P, None], (5, 7, 8, 9, 17)),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("off", [1, 2, 3])
def test_tables_off_a_multiple_of_four(name, off):
    args, tables = CALLS[name]
    for i in tables:
        call = list(args)
        call[i] = P + off
        assert getattr(_capi.lib(), name)(*call) == MISALIGNED, (name, i)
