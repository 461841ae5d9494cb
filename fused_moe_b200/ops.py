"""Operators beside the fused layer, for a user's own tensors: the activations' 8-bit format, the dense product in the experts'
weight format, and tokens sorted by expert and back.

    codes, scale = quantize(x)                        # what ``run`` takes as hidden_states, hidden_states_scale
    h = block_matmul(codes, scale, w, w_scale)        # [T, N], w [N, K] with 128x128 block scales like an expert's
    codes, scale = quantize(h, swiglu=True)           # silu gate between the two products of a feed-forward layer

    ids, weights = route(logits, bias, scaling)       # or any router's choice
    order = sort_tokens(ids)
    rows = permute(x, order)                          # differentiable
    out = unpermute(expert_rows, order, weights)      # differentiable in both

The layer from parts is the sequence route, sort_tokens, permute, quantize, block_matmul per expert, quantize with SwiGLU,
block_matmul, unpermute.  The step in the middle is the caller's: block_matmul takes one expert's rows, so the segments
(``order.offsets.tolist()``) have to be read on the host, which waits for the sort and cannot be captured (``run`` is the layer
without that).  Equal calls give equal results bit for bit (there are no atomics on values); calls of other sizes may add up in
another order (block_matmul's parts of K, see ``b200moe_block_matmul_form``, and the threads that sum a weight's gradient), so that a token's
last bits can differ between batch sizes.  Every call is asynchronous on the current stream of its tensors' device, can be captured
into a CUDA graph and allocates only its results (and the sort, above
16384 pairs, a scratch tensor) from torch's allocator.  Errors: ``TypeError`` / ``ValueError`` for arguments, ``RuntimeError``
for tensors that are not on one CUDA device, ``MoEError`` for what the library refuses, and at the next call of any operator on the
device after a ``block_matmul`` there gave up on a bounded wait (its result holds NaN then).  A replayed graph makes no call:
``check_status`` looks.  A backward pass is captured like any of
torch's: after a warm-up on a side stream, with no earlier graph of the same leaves alive (torch warns about its AccumulateGrad
node and the capture fails).  Gradients are first order and reverse mode: tensors with a forward-mode tangent are refused.

The reference has no counterparts: its only public function is the fused layer (solution/python/kernel.py:642-648).
"""
from __future__ import annotations

import ctypes as C
from typing import Dict, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _capi
from ._capi import MoEError
from .kernel import BLOCK, E_GLOBAL

_INT_MAX = 2 ** 31 - 1
_SORT_ONE_LAUNCH = 16384      # pairs that the sort handles without a scratch tensor
_CODES = (torch.float8_e4m3fn, torch.uint8)
_DTYPE = {torch.float32: _capi.F32, torch.bfloat16: _capi.BF16, torch.float16: _capi.F16}


# what a call asks of torch besides its tensors, without the Python layers above: half a microsecond instead of four (None where
# torch was built without CUDA, and with it any tensor that a call would take)
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


_functions: Dict[str, object] = {}


class _Status:
    """Pinned words of one device where a kernel that gave up on a bounded wait leaves its code."""

    def __init__(self, index: int):
        words = C.c_void_p()
        with torch.cuda.device(index):
            _capi.check(_capi.lib().b200moe_status_words(C.byref(words)), "b200moe_status_words")
        self.ptr = words.value
        self.view = (C.c_int32 * 4).from_address(self.ptr)

    def raise_if_failed(self) -> None:
        if self.view[0]:
            code, where = self.view[0], self.view[1]
            self.view[0] = 0
            raise MoEError(code, "device status of an earlier b200moe_block_matmul on this device", f"detail={where}")


_status: Dict[int, _Status] = {}


def check_status(device=None) -> None:
    """Waits for the device (None: the current one) and raises ``MoEError`` if a ``block_matmul`` on it gave up on a bounded wait
    since the last look, in a replayed graph too.  Such a product holds NaN where a sum was cut short."""
    dev = torch.device("cuda" if device is None else device)
    if dev.type != "cuda":
        raise RuntimeError(f"device is {dev}: fused_moe_b200 runs on CUDA devices only (there is no CPU path)")
    index = torch.cuda.current_device() if dev.index is None else dev.index
    torch.cuda.synchronize(index)
    st = _status.get(index)
    if st is not None:
        st.raise_if_failed()


def _call(name: str, index: int, *args) -> None:
    """Library call with its device current, on that device's current stream (the last argument).  What an earlier call there left
    in the status words is raised first."""
    st = _status.get(index)
    if st is not None and st.view[0]:
        st.raise_if_failed()
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_capi.lib(), name)
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _capi.check(rc, name)


def _not_cuda(t: torch.Tensor, what: str) -> RuntimeError:
    return RuntimeError(f"{what} is on {t.device}: fused_moe_b200 runs on CUDA tensors only (there is no CPU path)")


def _other_device(dev: torch.device, **tensors) -> RuntimeError:
    """The error for arguments of which one is not on ``dev``."""
    name, t = next((n, t) for n, t in tensors.items() if t is not None and t.device != dev)
    return RuntimeError(f"{name} is on {t.device}, the other arguments on {dev}")


def _no_gradient(what: str) -> RuntimeError:
    return RuntimeError(f"{what} has no gradient: detach its inputs or call it under torch.no_grad()")


def _refuse_duals(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Raises for a tensor with a forward-mode tangent, which a library call would drop without a word (it does not make
    ``requires_grad`` true).  Called only where a level of dual numbers is open."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative: detach its inputs")


def _matrix(t: torch.Tensor, what: str) -> Tuple[torch.Tensor, int, int, int]:
    """(``t``, rows, columns, row stride in elements) with unit inner stride, rows that do not overlap and values as they are stored (a
    copy where ``t`` has not: ``z.conj().imag`` is stored with the other sign); extents that 32 bits hold.  The stride of a single row is free: torch may say anything."""
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{what} must be 2-D, got shape {tuple(shape)}")
    rows, cols = shape
    if rows > _INT_MAX or cols > _INT_MAX:
        raise ValueError(f"{what} must have at most {_INT_MAX} rows and columns, got shape {tuple(shape)}")
    if t.is_neg():
        t = t.resolve_neg()
    if t.is_contiguous():
        return t, rows, cols, cols
    s0, s1 = t.stride()
    if (cols > 1 and s1 != 1) or (rows > 1 and s0 < cols):
        return t.contiguous(), rows, cols, cols
    return t, rows, cols, s0 if rows > 1 else cols


def _pitch(t: torch.Tensor) -> int:
    """Row stride in elements of a result that was checked."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check_out(out: torch.Tensor, shape: Tuple[int, ...], dtype: torch.dtype, dev: torch.device) -> None:
    if out.dtype != dtype or tuple(out.shape) != shape or out.device != dev:
        raise ValueError(f"out must be {dtype} {list(shape)} on {dev}, got {out.dtype} {list(out.shape)} on {out.device}")
    if (shape[1] > 1 and out.stride(1) != 1) or (shape[0] > 1 and out.stride(0) < shape[1]):
        raise ValueError("out must have unit inner stride and rows that do not overlap")
    if out.is_neg():
        raise ValueError("out must not be the imaginary part of a conjugate, which is stored with the other sign")
    if out.requires_grad:
        raise RuntimeError("out must not require a gradient")


def _written(out: torch.Tensor) -> None:
    """Tells autograd that ``out`` changed, as torch's own functions do: a graph that saved it refuses to go backward through it."""
    torch.autograd.graph.increment_version(out)


# ---- quantisation ----

def quantize(x: torch.Tensor, *, swiglu: bool = False, scale_layout: str = "kt") -> Tuple[torch.Tensor, torch.Tensor]:
    """Activations [T, K] (fp32, bf16 or fp16) as (e4m3 codes [T, K], fp32 scales of each 1x128 block).

    ``scale = max(max|x|, 1e-12) / 448`` per block, ``code = e4m3(x / scale)``, the quotient rounded to fp32 first: bit for bit
    ``synth.quant_rows_1x128``.  ``scale_layout`` "kt" gives the scales as [ceil(K/128), T], the layer's layout, "tk" as
    [T, ceil(K/128)].  With ``swiglu`` the input is [T, 2K] and what is quantised is ``x[:, :K] * silu(x[:, K:])`` in fp32
    (where ``silu`` of less than -88.7 is zero: 1 + exp(-u) is infinite).
    A block that holds an infinity or a NaN gets it as its scale, and codes as the quotient says.  Any K; not differentiable.
    """
    if not x.is_cuda:
        raise _not_cuda(x, "x")
    dev = x.device
    dt = _DTYPE.get(x.dtype)
    if dt is None:
        raise TypeError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    if scale_layout not in ("kt", "tk"):
        raise ValueError(f"scale_layout must be 'kt' or 'tk', got {scale_layout!r}")
    if x.requires_grad and torch.is_grad_enabled():
        raise _no_gradient("quantize")
    if forward_ad._current_level >= 0:
        _refuse_duals("quantize", x)
    x, rows, cols, pitch = _matrix(x, "x")
    if swiglu:
        if cols % 2:
            raise ValueError(f"swiglu needs an even number of columns (gate half, up half), got {cols}")
        cols //= 2
    blocks = -(-cols // BLOCK)
    codes = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device=dev)
    if scale_layout == "kt":
        scale, stride_t, stride_kb = torch.empty(blocks, rows, dtype=torch.float32, device=dev), 1, rows
    else:
        scale, stride_t, stride_kb = torch.empty(rows, blocks, dtype=torch.float32, device=dev), blocks, 1
    if rows and cols:
        _call("b200moe_quantize", dev.index, x.data_ptr(), dt, pitch, rows, cols, int(swiglu), codes.data_ptr(), cols,
              scale.data_ptr(), stride_t, stride_kb)
    return codes, scale


# ---- block-scaled product ----

def _block_scale_strides(scale: torch.Tensor, rows: int, blocks: int, layout: str, what: str) -> Tuple[int, int]:
    """(stride over rows, stride over K blocks) of a scale tensor, in elements."""
    if scale.dtype != torch.float32:
        raise TypeError(f"{what} must be float32, got {scale.dtype}")
    if layout == "kt":
        if scale.shape == (blocks, rows):
            return (1, rows) if scale.is_contiguous() else scale.stride()[::-1]
    elif scale.shape == (rows, blocks):
        return (blocks, 1) if scale.is_contiguous() else scale.stride()
    want = (blocks, rows) if layout == "kt" else (rows, blocks)
    raise ValueError(f"{what} has shape {tuple(scale.shape)}, expected {want} for scale_layout {layout!r}")


def block_matmul(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, *, scale_layout: str = "kt",
                 out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``a @ b.T`` of e4m3 matrices with block scales, accumulated in fp32: [M, N] in ``out_dtype`` (bf16, fp16, fp32).

    a [M, K] e4m3 (or its uint8 bits) with a_scale fp32 per 1x128, [ceil(K/128), M] (``scale_layout`` "kt") or
    [M, ceil(K/128)] ("tk"); b [N, K] e4m3 with b_scale fp32 [ceil(N/128), ceil(K/128)], the layout of an expert's weights.
    K must be a multiple of 16, M and N may be any.  Rows of ``a`` whose pitch is not a multiple of 16 bytes are copied; ``b``
    must have unit inner stride and such a pitch.  Scales may have any strides and values; the product of a row's and a block's is
    rounded to fp32 before it meets the sums.  ``out`` writes into a tensor of the caller's
    (which must not overlap the inputs).  Not differentiable: the operands are codes.
    """
    if not a.is_cuda:
        raise _not_cuda(a, "a")
    dev = a.device
    if a_scale.device != dev or b.device != dev or b_scale.device != dev:
        raise _other_device(dev, a_scale=a_scale, b=b, b_scale=b_scale)
    if (a_scale.requires_grad or b_scale.requires_grad or a.requires_grad or b.requires_grad) and torch.is_grad_enabled():
        raise _no_gradient("block_matmul")
    if forward_ad._current_level >= 0:
        _refuse_duals("block_matmul", a, a_scale, b, b_scale, out)
    if a.dtype not in _CODES or b.dtype not in _CODES:
        raise TypeError(f"a and b must be float8_e4m3fn (or its uint8 bit pattern), got {a.dtype} and {b.dtype}")
    a, M, K, a_pitch = _matrix(a, "a")
    b_shape = b.shape
    if len(b_shape) != 2 or b_shape[1] != K:
        raise ValueError(f"b must be [N, {K}], got {tuple(b_shape)}")
    N = b_shape[0]
    if N > _INT_MAX:
        raise ValueError(f"b must have at most {_INT_MAX} rows, got {N}")
    if K == 0 or K % 16:
        raise ValueError(f"K must be a positive multiple of 16, got {K}")
    if scale_layout not in ("kt", "tk"):
        raise ValueError(f"scale_layout must be 'kt' or 'tk', got {scale_layout!r}")
    blocks = -(-K // BLOCK)
    if a_scale.is_neg() or b_scale.is_neg():
        a_scale, b_scale = a_scale.resolve_neg(), b_scale.resolve_neg()
    as_m, as_kb = _block_scale_strides(a_scale, M, blocks, scale_layout, "a_scale")
    bs_n, bs_kb = _block_scale_strides(b_scale, -(-N // BLOCK), blocks, "tk", "b_scale")
    a_ptr, b_ptr = a.data_ptr(), b.data_ptr()
    b_pitch, b_step = (K, 1) if b.is_contiguous() else b.stride()
    if N == 1:
        b_pitch = K
    if (b_ptr | b_pitch) % 16 or b_pitch < K or b_step != 1:
        raise ValueError("b must have unit inner stride and rows on 16-byte boundaries")
    if (a_ptr | a_pitch) % 16:
        a = a.clone(memory_format=torch.contiguous_format)
        a_ptr, a_pitch = a.data_ptr(), K
    if out is None:
        dt, out_pitch = _DTYPE.get(out_dtype), N
        if dt is None:
            raise TypeError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
        out = torch.empty(M, N, dtype=out_dtype, device=dev)
    else:
        dt = _DTYPE.get(out.dtype)
        if dt is None:
            raise TypeError(f"out must be float32, bfloat16 or float16, got {out.dtype}")
        _check_out(out, (M, N), out.dtype, dev)
        out_pitch = _pitch(out)
        _written(out)
    if M == 0 or N == 0:
        return out
    st = _status.get(dev.index)
    if st is None:
        st = _status.setdefault(dev.index, _Status(dev.index))
    _call("b200moe_block_matmul", dev.index, a_ptr, a_pitch, a_scale.data_ptr(), as_m, as_kb, b_ptr, b_pitch, b_scale.data_ptr(),
          bs_n, bs_kb, M, N, K, out.data_ptr(), dt, out_pitch, st.ptr)
    return out


# ---- tokens sorted by expert and back ----

class TokenOrder:
    """What ``sort_tokens`` found; int32 tensors on the ids' device (views of one, made when they are asked for).

    offsets [e_local + 1]  first row of each local expert, the last: rows in use
    counts  [e_local]      pairs of each local expert
    pos     [T, top_k]     row of each (token, k), -1 where the expert is not local
    pair    [rows]         token * top_k + k of each row, -1 in padding and behind the last expert
    """

    __slots__ = ("tokens", "top_k", "rows", "e_local", "local_expert_offset", "align", "device", "_table", "_pos_at", "_pair_at", "_pointers")

    def __init__(self, device, tokens, top_k, rows, e_local, local_expert_offset, align):
        self.tokens, self.top_k, self.rows = tokens, top_k, rows
        self.e_local, self.local_expert_offset, self.align = e_local, local_expert_offset, align
        # offsets, counts, pos, pair: the latter two at multiples of 16 bytes
        self._pos_at = (2 * e_local + 4) // 4 * 4
        self._pair_at = self._pos_at + (tokens * top_k + 3) // 4 * 4
        self._own(torch.empty(self._pair_at + rows, dtype=torch.int32, device=device))

    def _own(self, table: torch.Tensor) -> None:
        """Takes the table, and from it the device and the addresses of pos, pair and offsets."""
        ptr = table.data_ptr()
        self._table, self.device = table, table.device
        self._pointers = ptr + 4 * self._pos_at, ptr + 4 * self._pair_at, ptr

    # a copied or unpickled order has a table of its own, elsewhere
    def __getstate__(self):
        return {name: getattr(self, name) for name in self.__slots__ if name not in ("device", "_pointers")}

    def __setstate__(self, state):
        for name, value in state.items():
            if name != "_table":
                setattr(self, name, value)
        self._own(state["_table"])

    @property
    def offsets(self) -> torch.Tensor:
        return self._table[:self.e_local + 1]

    @property
    def counts(self) -> torch.Tensor:
        return self._table[self.e_local + 1:2 * self.e_local + 1]

    @property
    def pos(self) -> torch.Tensor:
        return self._table.as_strided((self.tokens, self.top_k), (self.top_k, 1), self._pos_at)

    @property
    def pair(self) -> torch.Tensor:
        return self._table[self._pair_at:]


def sort_tokens(topk_ids: torch.Tensor, e_local: int = E_GLOBAL, local_expert_offset: int = 0, *, align: int = 1) -> TokenOrder:
    """Stable sort of the pairs (token, k) by expert; ids int32 or int64 [T, top_k], top_k at most 32.

    Experts [local_expert_offset, local_expert_offset + e_local) are local (at most 1024); pairs of others get no row, and an
    expert that a token names twice gets two.  Each expert's rows start on a multiple of ``align`` (128: a matrix tile).  The
    order has ``T * top_k`` rows and, with ``align``, room for the padding: how many are in use stays on the device.
    """
    if not topk_ids.is_cuda:
        raise _not_cuda(topk_ids, "topk_ids")
    dev = topk_ids.device
    if topk_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"topk_ids must be int32 or int64, got {topk_ids.dtype}")
    ids, tokens, top_k, pitch = _matrix(topk_ids, "topk_ids")
    e_local, off, align = int(e_local), int(local_expert_offset), int(align)
    if not 1 <= top_k <= 32:
        raise ValueError(f"topk_ids must have 1 to 32 columns, got {top_k}")
    if not 1 <= e_local <= 1024:
        raise ValueError(f"e_local must be 1 to 1024, got {e_local}")
    if not 0 <= off < 2 ** 30:
        raise ValueError(f"local_expert_offset must not be negative, got {off}")
    if not 1 <= align <= 65536:
        raise ValueError(f"align must be 1 to 65536, got {align}")
    pairs = tokens * top_k
    rows = -(-(pairs + (align - 1) * min(pairs, e_local)) // align) * align
    if rows >= 2 ** 31:
        raise ValueError(f"{rows} sorted rows: int32 tables name at most {2 ** 31 - 1}")
    order = TokenOrder(dev, tokens, top_k, rows, e_local, off, align)
    ws, ws_bytes = None, 0
    if pairs > _SORT_ONE_LAUNCH:
        ws_bytes = _capi.lib().b200moe_sort_workspace_bytes(tokens, top_k, e_local)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    pos, pair, offsets = order._pointers
    _call("b200moe_sort_tokens", dev.index, ids.data_ptr(), ids.element_size() * 8, pitch, tokens, top_k, e_local, off, align,
          offsets + 4 * (e_local + 1), offsets, pos, pair, rows, None if ws is None else ws.data_ptr(), ws_bytes)
    return order


def _permute(x: torch.Tensor, order: TokenOrder, out: Optional[torch.Tensor]) -> torch.Tensor:
    x, _, H, pitch = _matrix(x, "x")
    size, y, y_pitch = x.element_size(), out, H
    if out is None:
        y = torch.empty(order.rows, H, dtype=x.dtype, device=x.device)
    else:
        y_pitch = _pitch(out)
    _call("b200moe_permute_rows", order.device.index, x.data_ptr(), pitch * size, H * size, size, order.tokens, order.top_k,
          *order._pointers, order.e_local, order.rows, y.data_ptr(), y_pitch * size, int(out is None))
    if out is not None:
        _written(out)
    return y


def _unpermute(y: torch.Tensor, order: TokenOrder, weights: Optional[torch.Tensor], out: Optional[torch.Tensor]) -> torch.Tensor:
    y, _, H, pitch = _matrix(y, "y")
    w_ptr, w_pitch = None, 0
    if weights is not None:
        weights, _, _, w_pitch = _matrix(weights, "weights")
        w_ptr = weights.data_ptr()
    res, res_pitch = out, H
    if out is None:
        res = torch.empty(order.tokens, H, dtype=y.dtype, device=y.device)
    else:
        res_pitch = _pitch(out)
    _call("b200moe_unpermute_rows", order.device.index, y.data_ptr(), _DTYPE[y.dtype], pitch, order._pointers[0], w_ptr, w_pitch,
          order.tokens, order.top_k, H, res.data_ptr(), res_pitch)
    if out is not None:
        _written(out)
    return res


def _first_order(backward):
    """``once_differentiable`` where a graph of the gradient is asked for; elsewhere without what that wrapper takes (4 us).  A
    gradient that is a dual number is refused like an argument."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, grad):
        if forward_ad._current_level >= 0:
            _refuse_duals("the gradient", grad)
        return guarded(ctx, grad) if torch.is_grad_enabled() else backward(ctx, grad)
    return staticmethod(run)


class _Permute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order):
        ctx.order = order
        return _permute(x, order, None)

    @_first_order
    def backward(ctx, dy):
        return _unpermute(dy, ctx.order, None, None), None


class _Unpermute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, order, weights):
        ctx.order = order
        ctx.save_for_backward(y if weights is not None and weights.requires_grad else None, weights)
        ctx.y_like = (y.shape, y.dtype)
        return _unpermute(y, order, weights, None)

    @_first_order
    def backward(ctx, dout):
        order, (y, weights) = ctx.order, ctx.saved_tensors
        (rows, H), dtype = ctx.y_like
        dev = dout.device
        dout, _, _, d_pitch = _matrix(dout, "grad")
        dy = torch.empty(rows, H, dtype=dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = torch.empty(order.tokens, order.top_k, dtype=torch.float32, device=dev) if ctx.needs_input_grad[2] else None
        y_ptr, y_pitch, w_ptr, w_pitch = None, 0, None, 0
        if dw is not None:
            y, _, _, y_pitch = _matrix(y, "y")
            y_ptr = y.data_ptr()
        if weights is not None:
            weights, _, _, w_pitch = _matrix(weights, "weights")
            w_ptr = weights.data_ptr()
        pos, pair, offsets = order._pointers
        _call("b200moe_unpermute_grad", dev.index, dout.data_ptr(), _DTYPE[dtype], d_pitch, y_ptr, y_pitch, w_ptr, w_pitch, pos, pair,
              offsets, order.e_local, order.tokens, order.top_k, H, rows, None if dy is None else dy.data_ptr(), H,
              None if dw is None else dw.data_ptr())
        return dy, None, dw


def permute(x: torch.Tensor, order: TokenOrder, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of x [T, H] in the sorted order, [order.rows, H]: ``y[pos[t, k]] = x[t]``, zeros in padding rows.

    Any type of 1, 2 or 4 bytes an element (e4m3 codes and their "tk" scales among them).  Rows behind the last expert are
    zero too, except in an ``out`` of the caller's (which must not overlap x), where they stay as they were.  Differentiable for
    fp32, bf16 and fp16 x (without ``out``): ``dx[t]`` is the sum of dy over the token's rows, in fp32, rounded once.
    """
    if not x.is_cuda:
        raise _not_cuda(x, "x")
    dev = x.device
    if order.device != dev:
        raise _other_device(dev, order=order)
    if x.dim() != 2 or x.shape[0] != order.tokens:
        raise ValueError(f"x must be [{order.tokens}, H], got {tuple(x.shape)}")
    if x.element_size() not in (1, 2, 4) or x.is_complex():
        raise TypeError(f"x must have elements of 1, 2 or 4 bytes, got {x.dtype}")
    if forward_ad._current_level >= 0:
        _refuse_duals("permute", x, out)
    if x.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise RuntimeError("permute with out= has no gradient: detach x or leave out away")
        if x.dtype not in _DTYPE:
            raise TypeError(f"permute has no gradient for {x.dtype}")
        return _Permute.apply(x, order)
    if out is not None:
        _check_out(out, (order.rows, x.shape[1]), x.dtype, dev)
    return _permute(x, order, out)


def unpermute(y: torch.Tensor, order: TokenOrder, weights: Optional[torch.Tensor] = None, *,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Sums of each token's rows: ``out[t] = sum_k weights[t, k] * y[pos[t, k]]``, k ascending, fp32, rounded once to y's type.

    y [order.rows, H] fp32, bf16 or fp16; weights fp32 [T, top_k], or None for ones.  Choices that are not local add nothing (a
    token without any is zero) whatever their weight.  ``out`` must not overlap y.  Differentiable in y and weights (without
    ``out``): rows of dy that no pair takes are zero, dw is 0 where the expert is not local.
    """
    if not y.is_cuda:
        raise _not_cuda(y, "y")
    dev = y.device
    if order.device != dev or (weights is not None and weights.device != dev):
        raise _other_device(dev, order=order, weights=weights)
    if y.dtype not in _DTYPE:
        raise TypeError(f"y must be float32, bfloat16 or float16, got {y.dtype}")
    if y.dim() != 2 or y.shape[0] != order.rows:
        raise ValueError(f"y must be [{order.rows}, H], got {tuple(y.shape)}")
    if weights is not None:
        if weights.dtype != torch.float32:
            raise TypeError(f"weights must be float32, got {weights.dtype}")
        if tuple(weights.shape) != (order.tokens, order.top_k):
            raise ValueError(f"weights must be [{order.tokens}, {order.top_k}], got {tuple(weights.shape)}")
    if forward_ad._current_level >= 0:
        _refuse_duals("unpermute", y, weights, out)
    if torch.is_grad_enabled() and (y.requires_grad or (weights is not None and weights.requires_grad)):
        if out is not None:
            raise RuntimeError("unpermute with out= has no gradient: detach its inputs or leave out away")
        return _Unpermute.apply(y, order, weights)
    if out is not None:
        _check_out(out, (order.tokens, y.shape[1]), y.dtype, dev)
    return _unpermute(y, order, weights, out)
