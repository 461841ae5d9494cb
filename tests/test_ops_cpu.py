"""Refusals of the operators beside the layer that need no GPU: the C ABI's argument checks (which run before any CUDA call and
write nothing) and the Python entry points on CPU tensors."""
import ctypes as C

import pytest
import torch

import fused_moe_b200 as F
from fused_moe_b200 import _capi

INVALID, SHAPE, SPACE, MISALIGNED = -1, -2, -3, -6


@pytest.fixture(scope="module")
def mem():
    buf = C.create_string_buffer(1 << 16)
    return buf, (C.addressof(buf) + 255) // 256 * 256


def test_quantize_refusals(mem):
    f, p = _capi.lib().b200moe_quantize, mem[1]
    ok = [p, 1, 256, 4, 256, 0, p, 256, p, 1, 4, None]

    def call(**kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return f(*a)
    assert call(_0=None) == INVALID and call(_6=None) == INVALID and call(_8=None) == INVALID
    assert call(_1=3) == INVALID and call(_1=-1) == INVALID
    assert call(_3=-1) == INVALID and call(_4=-1) == INVALID
    assert call(_2=255) == INVALID and call(_7=255) == INVALID          # pitches shorter than a row
    assert call(_5=1) == INVALID                                        # swiglu: rows of 2 x 256 elements
    assert call(_0=p + 1) == MISALIGNED and call(_8=p + 2) == MISALIGNED
    assert call(_4=0x40000000, _2=1 << 40, _7=1 << 40) == SHAPE
    assert call(_3=0) == 0 and call(_4=0) == 0                          # nothing to do: nothing is touched


def test_block_matmul_refusals(mem):
    f, p = _capi.lib().b200moe_block_matmul, mem[1]
    #     a, pitch, sa, m, kb, b, pitch, sb, n, kb, M, N, K, out, dtype, pitch, status, stream
    ok = [p, 256, p, 1, 4, p, 256, p, 2, 1, 4, 8, 256, p, 1, 8, None, None]

    def call(**kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return f(*a)
    for i in (0, 2, 5, 7, 13):
        assert call(**{f"_{i}": None}) == INVALID, i
    assert call(_10=-1) == INVALID and call(_11=-1) == INVALID and call(_12=0) == INVALID and call(_14=3) == INVALID
    assert call(_12=200) == SHAPE                                       # K not a multiple of 16
    assert call(_1=240) == INVALID and call(_6=240) == INVALID and call(_15=7) == INVALID
    assert call(_1=264) == MISALIGNED and call(_6=264) == MISALIGNED
    assert call(_0=p + 8) == MISALIGNED and call(_5=p + 8) == MISALIGNED and call(_13=p + 1) == MISALIGNED
    assert call(_10=0x7fffffff) == SHAPE
    assert call(_10=0) == 0 and call(_11=0) == 0


def test_sort_refusals(mem):
    lib, p = _capi.lib(), mem[1]
    f = lib.b200moe_sort_tokens
    #     ids, bits, pitch, T, k, E, off, align, counts, offsets, pos, pair, rows, ws, ws_bytes, stream
    ok = [p, 32, 8, 4, 8, 16, 0, 1, p, p, p, p, 32, None, 0, None]

    def call(**kw):
        a = list(ok)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return f(*a)
    for i in (0, 8, 9, 10, 11):
        assert call(**{f"_{i}": None}) == INVALID, i
    assert call(_1=16) == INVALID and call(_2=7) == INVALID and call(_3=-1) == INVALID and call(_4=0) == INVALID
    assert call(_5=0) == INVALID and call(_6=-1) == INVALID and call(_7=0) == INVALID
    assert call(_4=33, _2=33) == SHAPE and call(_5=1025) == SHAPE and call(_7=65537) == SHAPE
    assert call(_12=31) == SHAPE                                        # too few rows
    assert call(_3=1 << 31) == SHAPE
    assert call(_0=p + 4, _1=64) == MISALIGNED and call(_0=p + 2) == MISALIGNED
    assert lib.b200moe_sort_rows(4, 8, 16, 1) == 32
    assert lib.b200moe_sort_rows(4, 8, 16, 128) == -(-(32 + 127 * 16) // 128) * 128
    assert lib.b200moe_sort_rows(1, 2, 16, 128) == 256                  # two pairs: two segments at most
    assert lib.b200moe_sort_rows(0, 2, 16, 128) == 0
    assert lib.b200moe_sort_rows(4, 33, 16, 1) == INVALID and lib.b200moe_sort_rows(4, 8, 0, 1) == INVALID
    assert lib.b200moe_sort_workspace_bytes(4, 8, 0) == INVALID and lib.b200moe_sort_workspace_bytes(4, 33, 8) == INVALID
    # none up to the pairs that one launch sorts (the host allocates none either), then a histogram for each chunk
    assert lib.b200moe_sort_workspace_bytes(2048, 8, 256) == 0 and F.ops._SORT_ONE_LAUNCH == 2048 * 8
    assert lib.b200moe_sort_workspace_bytes(2049, 8, 256) == 10 * 256 * 4
    assert lib.b200moe_sort_workspace_bytes(65537, 8, 10) == (-(-65537 * 8 // 2048) + 1) * 10 * 4
    assert call(_3=3000, _12=24000) == INVALID and call(_3=3000, _12=24000, _13=p, _14=12 * 16 * 4 - 1) == SPACE


def test_row_moves_refusals(mem):
    lib, p = _capi.lib(), mem[1]
    #       x, pitch, bytes, elem, T, k, pos, pair, offsets, E, rows, y, pitch, zero, stream
    move = [p, 512, 512, 2, 4, 8, p, p, p, 16, 32, p, 512, 1, None]
    #      y, dtype, pitch, pos, w, pitch, T, k, H, out, pitch, stream
    back = [p, 1, 256, p, p, 8, 4, 8, 256, p, 256, None]
    #       dout, dtype, pitch, y, pitch, w, pitch, pos, pair, offsets, E, T, k, H, rows, dy, pitch, dw, stream
    grad = [p, 1, 256, p, 256, p, 8, p, p, p, 16, 4, 8, 256, 32, p, 256, p, None]

    def call(f, base, **kw):
        a = list(base)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return f(*a)
    f = lib.b200moe_permute_rows
    for i in (0, 6, 7, 8, 11):
        assert call(f, move, **{f"_{i}": None}) == INVALID, i
    assert call(f, move, _3=8) == INVALID and call(f, move, _2=511) == INVALID and call(f, move, _1=510) == INVALID
    assert call(f, move, _12=510) == INVALID and call(f, move, _5=33) == SHAPE and call(f, move, _0=p + 1) == MISALIGNED
    assert call(f, move, _1=513) == MISALIGNED and call(f, move, _10=0) == 0 and call(f, move, _2=0) == 0
    f = lib.b200moe_unpermute_rows
    for i in (0, 3, 9):
        assert call(f, back, **{f"_{i}": None}) == INVALID, i
    assert call(f, back, _1=5) == INVALID and call(f, back, _2=255) == INVALID and call(f, back, _10=255) == INVALID
    assert call(f, back, _5=7) == INVALID and call(f, back, _0=p + 1) == MISALIGNED and call(f, back, _6=0) == 0
    f = lib.b200moe_unpermute_grad
    for i in (0, 3, 7, 8, 9):
        assert call(f, grad, **{f"_{i}": None}) == INVALID, i
    assert call(f, grad, _1=5) == INVALID and call(f, grad, _2=255) == INVALID and call(f, grad, _16=255) == INVALID
    assert call(f, grad, _6=7) == INVALID and call(f, grad, _15=p + 1) == MISALIGNED
    assert call(f, grad, _15=None, _17=None) == 0


def test_python_entry_points_refuse_cpu_tensors():
    x = torch.zeros(4, 256)
    ids = torch.zeros(4, 8, dtype=torch.int32)
    order = F.TokenOrder(x.device, 4, 8, 32, 16, 0, 1)
    codes = torch.zeros(4, 256, dtype=torch.uint8)
    for call in (lambda: F.quantize(x), lambda: F.sort_tokens(ids), lambda: F.permute(x, order),
                 lambda: F.unpermute(torch.zeros(32, 256), order), lambda: F.block_matmul(codes, x, codes, x)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
