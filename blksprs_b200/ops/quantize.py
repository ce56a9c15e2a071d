"""8-bit values with a scale for each block of 128: the operands of ``grouped_matmul_scaled``.

``scale = max(largest magnitude of the block / largest value of the type, 2**-126)`` (the quotient as a product with the
rounded reciprocal, as torch divides by a number), ``q = value / scale`` rounded to nearest even; -0 stays -0.  A block
that holds an infinity or a NaN has a scale that is not finite and multiplies out to NaN; other blocks are not touched by
it.  No counterpart in the blksprs library.
"""
from __future__ import annotations

import torch
from torch import Tensor

from .. import _cabi
from ..utils.tools import plain_dispatch
from ..utils.validation import contiguous_enabled
from .grouped_matmul import SCALE_BLOCK, check_device, check_dimensions, check_no_tangents, forward_mode


def _validate(t: Tensor, dtype: torch.dtype, dims: int) -> None:
    if dtype not in _cabi.EIGHT_BIT_DTYPE_CODES:
        raise ValueError("Output dtype must be float8_e4m3fn or float8_e5m2")
    check_dimensions(dims, t)
    if t.dtype not in _cabi.DATA_DTYPE_CODES:
        raise ValueError("Tensor must have either float16, bfloat16, or float32 dtype")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("Rounding to 8 bits has no gradient")
    if forward_mode():
        check_no_tangents(t)
    check_device(t)


def _quantize_rows_eager(x: Tensor, dtype: torch.dtype) -> tuple[Tensor, Tensor]:
    _validate(x, dtype, 2)
    rows, width = x.shape
    if x.stride(1) != 1 and width > 1:
        if not contiguous_enabled():
            raise ValueError("Tensor must be contiguous")
        x = x.contiguous()
    device = x.device
    if _cabi.current_device() != device.index:
        with torch.cuda.device(device):
            return _quantize_rows_eager(x, dtype)
    q = x.new_empty((rows, width), dtype=dtype)
    scale = x.new_empty((rows, -(-width // SCALE_BLOCK)), dtype=torch.float32)
    status = _cabi.lib().bsp_quantize_rows(
        x.data_ptr(), x.stride(0), rows, width, _cabi.DATA_DTYPE_CODES[x.dtype], q.data_ptr(),
        _cabi.EIGHT_BIT_DTYPE_CODES[dtype], scale.data_ptr(), _cabi.stream_handle(device))
    if status:
        _cabi.check(status, "bsp_quantize_rows")
    return q, scale


def _quantize_blocks_eager(w: Tensor, dtype: torch.dtype) -> tuple[Tensor, Tensor]:
    _validate(w, dtype, 3)
    groups, depth, cols = w.shape
    device = w.device
    with _cabi.device_guard(device):
        q = torch.empty((groups, cols, depth), dtype=dtype, device=device).transpose(1, 2)
        scale = torch.empty((groups, -(-depth // SCALE_BLOCK), -(-cols // SCALE_BLOCK)), dtype=torch.float32,
                            device=device)
        _cabi.check(_cabi.lib().bsp_quantize_blocks(
            w.data_ptr(), *w.stride(), groups, depth, cols, _cabi.DATA_DTYPE_CODES[w.dtype], q.data_ptr(),
            _cabi.EIGHT_BIT_DTYPE_CODES[dtype], scale.data_ptr(), _cabi.stream_handle(device)), "bsp_quantize_blocks")
    return q, scale


# What a compiled caller calls, so that the rounding stays inside its graph.

@torch.library.custom_op("blksprs_b200::quantize_rows", mutates_args=(), device_types="cuda")
def _registered_rows(x: Tensor, dtype: torch.dtype) -> tuple[Tensor, Tensor]:
    return _quantize_rows_eager(x, dtype)


@_registered_rows.register_fake
def _(x, dtype):
    return (x.new_empty((x.size(0), x.size(1)), dtype=dtype),
            x.new_empty((x.size(0), (x.size(1) + SCALE_BLOCK - 1) // SCALE_BLOCK), dtype=torch.float32))


@torch.library.custom_op("blksprs_b200::quantize_blocks", mutates_args=(), device_types="cuda")
def _registered_blocks(w: Tensor, dtype: torch.dtype) -> tuple[Tensor, Tensor]:
    """The matrices as they are stored: (groups, columns, depth)."""
    q, scale = _quantize_blocks_eager(w, dtype)
    return q.transpose(1, 2), scale


@_registered_blocks.register_fake
def _(w, dtype):
    return (w.new_empty((w.size(0), w.size(2), w.size(1)), dtype=dtype),
            w.new_empty((w.size(0), (w.size(1) + SCALE_BLOCK - 1) // SCALE_BLOCK,
                         (w.size(2) + SCALE_BLOCK - 1) // SCALE_BLOCK), dtype=torch.float32))


_quantize_rows_plain = plain_dispatch(_quantize_rows_eager)
_quantize_blocks_plain = plain_dispatch(_quantize_blocks_eager)
_quantize_rows_no_compile = torch.compiler.disable(_quantize_rows_plain)
_quantize_blocks_no_compile = torch.compiler.disable(_quantize_blocks_plain)


def _in_graph(t: Tensor) -> bool:
    """Whether a compiled call becomes part of the caller's graph; others break it (and are refused where they have to be)."""
    return (type(t) in (Tensor, torch.nn.Parameter) and not (t.requires_grad and torch.is_grad_enabled())
            and not forward_mode())


def quantize_rows(x: Tensor, dtype: torch.dtype = torch.float8_e4m3fn) -> tuple[Tensor, Tensor]:
    """Rounds rows to 8 bits with a scale for each 128 neighbouring values of a row.

    Args:
        x (Tensor): The rows ``(T, K)``, float16, bfloat16 or float32; the last block of a row may be short.
        dtype (torch.dtype): float8_e4m3fn (default) or float8_e5m2.

    Returns:
        tuple[Tensor, Tensor]: The rounded rows ``(T, K)`` and the scales, float32 ``(T, ceil(K / 128))``.
    """
    if torch.compiler.is_compiling():
        return (_registered_rows if _in_graph(x) else _quantize_rows_no_compile)(x, dtype)
    return (_quantize_rows_eager if type(x) is Tensor else _quantize_rows_plain)(x, dtype)


def quantize_blocks(w: Tensor, dtype: torch.dtype = torch.float8_e4m3fn) -> tuple[Tensor, Tensor]:
    """Rounds matrices to 8 bits with a scale for each block of 128 x 128.

    Args:
        w (Tensor): One matrix per group ``(E, K, N)``, float16, bfloat16 or float32, any strides; the blocks at the
            edges may be smaller.
        dtype (torch.dtype): float8_e4m3fn (default) or float8_e5m2.

    Returns:
        tuple[Tensor, Tensor]: The rounded matrices ``(E, K, N)``, stored with ``K`` contiguous as
        ``grouped_matmul_scaled`` reads them, and the scales, float32 ``(E, ceil(K / 128), ceil(N / 128))``.
    """
    if torch.compiler.is_compiling():
        if not _in_graph(w):
            return _quantize_blocks_no_compile(w, dtype)
        q, scale = _registered_blocks(w, dtype)
        return q.transpose(1, 2), scale
    return (_quantize_blocks_eager if type(w) is Tensor else _quantize_blocks_plain)(w, dtype)
