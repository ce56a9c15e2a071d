"""Matrix products grouped by expert, in 16 bits with gradients and in 8 bits with block scales.

The rows of ``x`` are sorted by group; ``group_offsets`` (on the device) says where each group's rows begin and end.
A layer of experts is a block-sparse product whose row blocks have any height: where ``matmul`` takes a layout of
equal blocks, the functions here take the group bounds, so no row is padded to a block and no layout is rebuilt when
the router sends the next batch elsewhere.  The group bounds are never read back to the host; all calls can be
recorded into a CUDA graph and replayed with other bounds in the same tensor.

No counterpart in the blksprs library.
"""
from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import forward_ad

from .. import _cabi
from ..plan import status_word
from ..utils.tools import cast_for_autocast, plain_dispatch
from ..utils.validation import contiguous_enabled

_16_BIT = {t: _cabi.DATA_DTYPE_CODES[t] for t in (torch.float16, torch.bfloat16)}
_8_BIT = _cabi.EIGHT_BIT_DTYPE_CODES
_INDEX_DTYPES = (torch.int32, torch.int64)
_OUT_DTYPES = {t: _cabi.DATA_DTYPE_CODES[t] for t in (torch.float16, torch.bfloat16, torch.float32)}
SCALE_BLOCK = 128
MAX_GROUPS = 1024


# The checks below do not go by the validation switch: they read nothing from the device and cost a microsecond or
# two, and operands that do not fit together would be read out of bounds.

def check_dimensions(dims: int, *tensors: Tensor) -> None:
    if any(t.dim() != dims for t in tensors):
        raise ValueError(f"Tensor must have {dims} dimensions")


def check_device(*tensors: Tensor) -> None:
    if tensors[0].device.type != "cuda":
        raise ValueError("Tensors must be on GPU")
    if any(t.device != tensors[0].device for t in tensors[1:]):
        raise ValueError("Tensors must be on same device")


def forward_mode() -> bool:
    """Whether a forward-mode level is open (one attribute; a torch without it looks at the tensors every time)."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def check_no_tangents(*tensors: Tensor) -> None:
    """A tangent would be lost without a word: a dual tensor need not require a gradient."""
    if any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError("Forward-mode gradients are not supported")


def _copied(t: Tensor, in_backward: bool = False) -> Tensor:
    if not (in_backward or contiguous_enabled()):
        raise ValueError("Tensor must be contiguous")
    return t.clone(memory_format=torch.contiguous_format)


# What the kernels read in place: rows, and matrices with either of their dimensions contiguous, that start on 16-byte
# boundaries; anything else is copied.  (A call on a few rows takes the GPU about as long as Python takes for a few dozen
# of its steps, so these and the checks are written as straight lines.)

def _row_stride(t: Tensor, mask: int) -> int:
    """Row stride of ``t`` (rows, width) if it is read in place, else 0; ``mask`` = elements of 16 bytes, less one."""
    ld, inner = t.stride()
    if inner != 1 or t.data_ptr() & 15:
        return 0
    rows, width = t.shape
    if rows == 1:
        return width
    return 0 if ld < width or ld & mask else ld


def _group_and_outer_stride(w: Tensor, mask: int) -> tuple[int, int, bool]:
    """Group stride, stride of the outer matrix dimension and whether the columns are the inner one, of ``w``
    (groups, depth, columns) if it is read in place; else the second is 0."""
    sg, sk, sn = w.stride()
    groups, depth, cols = w.shape
    if groups == 1:
        sg = depth * cols
    elif sg <= mask or sg & mask:
        return sg, 0, True
    if not w.data_ptr() & 15:
        if sn == 1 and sk >= cols and not sk & mask:
            return sg, sk, True
        if sk == 1 and sn >= depth and not sn & mask:
            return sg, sn, False
    return sg, 0, True


def _validate_offsets(group_offsets: Tensor, groups: int) -> None:
    if group_offsets.dtype not in (torch.int32, torch.int64):
        raise ValueError("Group offsets must have either int32 or int64 dtype")
    if group_offsets.dim() != 1 or group_offsets.size(0) != groups + 1:
        raise ValueError("Group offsets must have one entry more than there are groups")
    if not group_offsets.is_contiguous():
        raise ValueError("Tensor must be contiguous")


def _validate_groups(x: Tensor, w: Tensor, group_offsets: Tensor, vector: int) -> None:
    _validate_offsets(group_offsets, w.size(0))
    if x.size(1) != w.size(1):
        raise ValueError("Inner dimensions of tensors must match")
    if w.size(0) > MAX_GROUPS:
        raise ValueError(f"Number of groups must be at most {MAX_GROUPS}")
    if x.size(1) % vector or w.size(2) % 8:
        raise ValueError(f"Inner dimension must be divisible by {vector} and columns by 8")


def _validate(x: Tensor, w: Tensor, group_offsets: Tensor) -> None:
    x_shape, w_shape, dtype, device = x.shape, w.shape, x.dtype, x.device
    # all at once; which one it was is sorted out only if this fails
    if len(x_shape) == 2 and len(w_shape) == 3:
        groups, depth, cols = w_shape
        if (x_shape[1] == depth and dtype in _16_BIT and w.dtype is dtype and groups <= MAX_GROUPS and not depth & 7
                and not cols & 7 and group_offsets.dtype in _INDEX_DTYPES and group_offsets.shape == (groups + 1,)
                and group_offsets.is_contiguous() and device.type == "cuda" and w.device == device
                and group_offsets.device == device):
            return
    check_dimensions(2, x)
    check_dimensions(3, w)
    if x.dtype not in _16_BIT:
        raise ValueError("Tensor must have either float16 or bfloat16 dtype")
    if w.dtype != x.dtype:
        raise ValueError("Tensors must have same dtype")
    _validate_groups(x, w, group_offsets, 8)
    check_device(x, w, group_offsets)


def _validate_gradient(x: Tensor, grad: Tensor, group_offsets: Tensor) -> None:
    check_dimensions(2, x, grad)
    if x.dtype not in _16_BIT:
        raise ValueError("Tensor must have either float16 or bfloat16 dtype")
    if grad.dtype != x.dtype:
        raise ValueError("Tensors must have same dtype")
    if grad.size(0) != x.size(0):
        raise ValueError("Numbers of rows must match")
    groups = max(group_offsets.numel() - 1, 0)
    _validate_offsets(group_offsets, groups)
    if groups > MAX_GROUPS:
        raise ValueError(f"Number of groups must be at most {MAX_GROUPS}")
    if x.size(1) % 8 or grad.size(1) % 8:
        raise ValueError("Inner dimension must be divisible by 8 and columns by 8")
    check_device(x, grad, group_offsets)


def _rows_product(x: Tensor, w: Tensor, group_offsets: Tensor, in_backward: bool = False) -> Tensor:
    """``out[t] = x[t] @ w[group of t]``, zero for rows of no group."""
    rows, depth = x.shape
    groups, _, cols = w.shape
    device = x.device
    if not (rows and cols and depth and groups):
        return torch.zeros((rows, cols), dtype=x.dtype, device=device)
    if _cabi.current_device() != device.index:
        with torch.cuda.device(device):
            return _rows_product(x, w, group_offsets, in_backward)
    ld_x = _row_stride(x, 7)
    if not ld_x:
        x, ld_x = _copied(x, in_backward), depth
    group_stride, ld_w, columns_inner = _group_and_outer_stride(w, 7)
    if not ld_w:
        w, group_stride, ld_w, columns_inner = _copied(w, in_backward), depth * cols, cols, True
    out = x.new_empty((rows, cols))
    status = _cabi.lib().bsp_grouped_matmul(
        x.data_ptr(), ld_x, w.data_ptr(), group_stride, ld_w, columns_inner, group_offsets.data_ptr(),
        group_offsets.dtype is torch.int64, rows, groups, depth, cols, out.data_ptr(), _16_BIT[x.dtype],
        status_word(device).data_ptr(), _cabi.stream_handle(device))
    if status:
        _cabi.check(status, "bsp_grouped_matmul")
    return out


def _weight_gradient(x: Tensor, grad: Tensor, group_offsets: Tensor, groups: int) -> Tensor:
    """``out[e] = x[rows of e]^T @ grad[rows of e]``, zero for groups without rows."""
    rows, depth = x.shape
    cols = grad.size(1)
    device = x.device
    if not (rows and cols and depth and groups):
        return torch.zeros((groups, depth, cols), dtype=x.dtype, device=device)
    if _cabi.current_device() != device.index:
        with torch.cuda.device(device):
            return _weight_gradient(x, grad, group_offsets, groups)
    ld_x, ld_grad = _row_stride(x, 7), _row_stride(grad, 7)
    if not ld_x:
        x, ld_x = _copied(x, True), depth
    if not ld_grad:
        grad, ld_grad = _copied(grad, True), cols
    out = x.new_empty((groups, depth, cols))
    lib = _cabi.lib()
    size = lib.bsp_grouped_weight_grad_workspace(rows, groups, depth, cols)
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    status = lib.bsp_grouped_weight_grad(
        x.data_ptr(), ld_x, grad.data_ptr(), ld_grad, group_offsets.data_ptr(), group_offsets.dtype is torch.int64,
        rows, groups, depth, cols, out.data_ptr(), _16_BIT[x.dtype], workspace.data_ptr() if size else None, size,
        status_word(device).data_ptr(), _cabi.stream_handle(device))
    if status:
        _cabi.check(status, "bsp_grouped_weight_grad")
    return out


class _GroupedMatmul(torch.autograd.Function):
    """Differentiable in ``x`` and ``w``: dX = dO W^T (the same rows product), dW = X^T dO by group."""

    @staticmethod
    def forward(ctx, x: Tensor, w: Tensor, group_offsets: Tensor):
        ctx.save_for_backward(x, w, group_offsets)
        return _rows_product(x, w, group_offsets)

    @staticmethod
    @torch.autograd.function.once_differentiable
    @plain_dispatch
    def backward(ctx, grad_output: Tensor):
        x, w, group_offsets = ctx.saved_tensors
        if forward_mode():
            check_no_tangents(grad_output)
        if grad_output.dtype != x.dtype:
            grad_output = grad_output.to(x.dtype)
        grad_x = grad_w = None
        if ctx.needs_input_grad[0]:
            grad_x = _rows_product(grad_output, w.transpose(1, 2), group_offsets, True)
        if ctx.needs_input_grad[1]:
            if w.stride(1) == 1 and w.stride(2) != 1:
                # weights stored with the depth innermost get their gradient in the same order
                grad_w = _weight_gradient(grad_output, x, group_offsets, w.size(0)).transpose(1, 2)
            else:
                grad_w = _weight_gradient(x, grad_output, group_offsets, w.size(0))
        return grad_x, grad_w, None


def _grouped_matmul_eager(x, w, group_offsets):
    if torch.is_autocast_enabled():
        x, w = cast_for_autocast(x, w)
    if forward_mode():
        check_no_tangents(x, w)
    _validate(x, w, group_offsets)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        return _GroupedMatmul.apply(x, w, group_offsets)
    return _rows_product(x, w, group_offsets)


# What a compiled caller calls: the same launches as registered ops, so that they stay inside its graph.  In the backward
# pass the operands are copied where they have to be, whatever the switch for inputs says.

@torch.library.custom_op("blksprs_b200::grouped_matmul", mutates_args=(), device_types="cuda")
def _registered_product(x: Tensor, w: Tensor, group_offsets: Tensor, in_backward: bool = False) -> Tensor:
    if forward_mode():
        check_no_tangents(x, w)
    _validate(x, w, group_offsets)
    return _rows_product(x, w, group_offsets, in_backward)


@_registered_product.register_fake
def _(x, w, group_offsets, in_backward=False):
    return x.new_empty((x.size(0), w.size(2)))


@torch.library.custom_op("blksprs_b200::grouped_weight_gradient", mutates_args=(), device_types="cuda")
def _registered_weight_gradient(x: Tensor, grad: Tensor, group_offsets: Tensor) -> Tensor:
    if forward_mode():
        check_no_tangents(x, grad)
    _validate_gradient(x, grad, group_offsets)
    return _weight_gradient(x, grad, group_offsets, group_offsets.size(0) - 1)


@_registered_weight_gradient.register_fake
def _(x, grad, group_offsets):
    return x.new_empty((group_offsets.size(0) - 1, x.size(1), grad.size(1)))


def _registered_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:3])


def _registered_backward(ctx, grad_output):
    x, w, group_offsets = ctx.saved_tensors
    grad_x = grad_w = None
    if ctx.needs_input_grad[0]:
        grad_x = _registered_product(grad_output, w.transpose(1, 2), group_offsets, True)
    if ctx.needs_input_grad[1]:
        if w.stride(1) == 1 and w.stride(2) != 1:
            grad_w = _registered_weight_gradient(grad_output, x, group_offsets).transpose(1, 2)
        else:
            grad_w = _registered_weight_gradient(x, grad_output, group_offsets)
    return grad_x, grad_w, None, None


_registered_product.register_autograd(_registered_backward, setup_context=_registered_setup)

_PLAIN = (Tensor, torch.nn.Parameter)
_grouped_matmul_plain = plain_dispatch(_grouped_matmul_eager)
_grouped_matmul_no_compile = torch.compiler.disable(_grouped_matmul_plain)


def grouped_matmul(x: Tensor, w: Tensor, group_offsets: Tensor) -> Tensor:
    """Multiplies the rows of every group with that group's matrix.

    ``out[t] = x[t] @ w[e]`` for ``group_offsets[e] <= t < group_offsets[e + 1]``; rows of no group (before the
    first offset, behind the last) are zero, and so are their gradients and the gradient of a group without rows.
    Sums run in float32 and are rounded once. Forward-mode gradients are refused.

    Args:
        x (Tensor): The rows ``(T, K)``, sorted by group, float16 or bfloat16. ``K`` is a multiple of 8.
        w (Tensor): One matrix per group ``(E, K, N)``, same dtype, ``E <= 1024``, ``N`` a multiple of 8. Either of
            the last two dimensions may be the contiguous one (``linear_weights.transpose(1, 2)`` is not copied).
        group_offsets (Tensor): int32 or int64 ``(E + 1,)`` on the device, non-decreasing, within ``0 .. T``. The
            values are not read by the host: ones that break this are clamped on the device and reported by
            ``plan.check_device_status``.

    Returns:
        Tensor: The products ``(T, N)``.
    """
    if torch.compiler.is_compiling():
        if type(x) not in _PLAIN or type(w) not in _PLAIN or forward_mode():
            return _grouped_matmul_no_compile(x, w, group_offsets)
        if torch.is_autocast_enabled():
            x, w = cast_for_autocast(x, w)
        return _registered_product(x, w, group_offsets)
    # only other tensor subclasses need their dispatch switched off
    impl = _grouped_matmul_eager if type(x) in _PLAIN and type(w) in _PLAIN else _grouped_matmul_plain
    return impl(x, w, group_offsets)


def _blocks_of(size: int) -> int:
    return -(-size // SCALE_BLOCK)


def _validate_scaled(x, scale_x, w, scale_w, group_offsets, out_dtype) -> None:
    if out_dtype not in _OUT_DTYPES:
        raise ValueError("Output dtype must be float16, bfloat16, or float32")
    x_shape, w_shape, device = x.shape, w.shape, x.device
    if len(x_shape) == 2 and len(w_shape) == 3:
        groups, depth, cols = w_shape
        blocks = -(-depth // SCALE_BLOCK)
        if (x_shape[1] == depth and x.dtype in _8_BIT and w.dtype in _8_BIT and groups <= MAX_GROUPS
                and not depth & 15 and not cols & 7 and scale_x.dtype is torch.float32
                and scale_w.dtype is torch.float32 and scale_x.shape == (x_shape[0], blocks)
                and scale_w.shape == (groups, blocks, -(-cols // SCALE_BLOCK))
                and group_offsets.dtype in _INDEX_DTYPES and group_offsets.shape == (groups + 1,)
                and group_offsets.is_contiguous() and device.type == "cuda" and w.device == device
                and scale_x.device == device and scale_w.device == device and group_offsets.device == device
                and not ((scale_x.requires_grad or scale_w.requires_grad or x.requires_grad or w.requires_grad)
                         and torch.is_grad_enabled())):
            return
    check_dimensions(2, x, scale_x)
    check_dimensions(3, w, scale_w)
    for t in (x, w):
        if t.dtype not in _cabi.EIGHT_BIT_DTYPE_CODES:
            raise ValueError("Tensor must have either float8_e4m3fn or float8_e5m2 dtype")
    for t in (scale_x, scale_w):
        if t.dtype != torch.float32:
            raise ValueError("Tensor must have float32 dtype")
    _validate_groups(x, w, group_offsets, 16)
    if tuple(scale_x.shape) != (x.size(0), _blocks_of(x.size(1))):
        raise ValueError(f"Scale shape {tuple(scale_x.shape)} doesn't match expected "
                         f"{(x.size(0), _blocks_of(x.size(1)))}")
    expected = (w.size(0), _blocks_of(w.size(1)), _blocks_of(w.size(2)))
    if tuple(scale_w.shape) != expected:
        raise ValueError(f"Scale shape {tuple(scale_w.shape)} doesn't match expected {expected}")
    if torch.is_grad_enabled() and (scale_x.requires_grad or scale_w.requires_grad or x.requires_grad
                                    or w.requires_grad):
        raise ValueError("The scaled product has no gradient")
    check_device(x, scale_x, w, scale_w, group_offsets)


def _grouped_matmul_scaled_eager(x, scale_x, w, scale_w, group_offsets, out_dtype):
    if forward_mode():
        check_no_tangents(x, scale_x, w, scale_w)
    _validate_scaled(x, scale_x, w, scale_w, group_offsets, out_dtype)
    return _scaled_product(x, scale_x, w, scale_w, group_offsets, out_dtype)


def _scaled_product(x, scale_x, w, scale_w, group_offsets, out_dtype):
    rows, depth = x.shape
    groups, _, cols = w.shape
    device = x.device
    if not (rows and cols and depth and groups):
        return torch.zeros((rows, cols), dtype=out_dtype, device=device)
    if _cabi.current_device() != device.index:
        with torch.cuda.device(device):
            return _scaled_product(x, scale_x, w, scale_w, group_offsets, out_dtype)
    ld_x = _row_stride(x, 15)
    if not ld_x:
        x, ld_x = _copied(x), depth
    group_stride, ld_w, columns_inner = _group_and_outer_stride(w, 15)
    if not ld_w or columns_inner:
        w, group_stride, ld_w = _copied(w.transpose(1, 2)).transpose(1, 2), depth * cols, depth
    out = x.new_empty((rows, cols), dtype=out_dtype)
    status = _cabi.lib().bsp_grouped_matmul_scaled(
        x.data_ptr(), ld_x, _8_BIT[x.dtype], scale_x.data_ptr(), *scale_x.stride(), w.data_ptr(), group_stride, ld_w,
        _8_BIT[w.dtype], scale_w.data_ptr(), *scale_w.stride(), group_offsets.data_ptr(),
        group_offsets.dtype is torch.int64, rows, groups, depth, cols, out.data_ptr(), _OUT_DTYPES[out_dtype],
        status_word(device).data_ptr(), _cabi.stream_handle(device))
    if status:
        _cabi.check(status, "bsp_grouped_matmul_scaled")
    return out


@torch.library.custom_op("blksprs_b200::grouped_matmul_scaled", mutates_args=(), device_types="cuda")
def _registered_scaled(x: Tensor, scale_x: Tensor, w: Tensor, scale_w: Tensor, group_offsets: Tensor,
                       out_dtype: torch.dtype) -> Tensor:
    return _grouped_matmul_scaled_eager(x, scale_x, w, scale_w, group_offsets, out_dtype)


@_registered_scaled.register_fake
def _(x, scale_x, w, scale_w, group_offsets, out_dtype):
    return x.new_empty((x.size(0), w.size(2)), dtype=out_dtype)


_grouped_matmul_scaled_plain = plain_dispatch(_grouped_matmul_scaled_eager)
_grouped_matmul_scaled_no_compile = torch.compiler.disable(_grouped_matmul_scaled_plain)


def grouped_matmul_scaled(x: Tensor, scale_x: Tensor, w: Tensor, scale_w: Tensor, group_offsets: Tensor,
                          out_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """:func:`grouped_matmul` of 8-bit operands that carry a scale for each block of 128.

    ``out[t, n] = sum over b of scale_x[t, b] * scale_w[e, b, n // 128] * (x[t, block b] . w[e, block b, n])``, the
    operands :func:`quantize_rows` and :func:`quantize_blocks` make. One group (``group_offsets = [0, T]``) is a
    linear layer. Every sum is float32, the result is rounded once. No gradient.

    Args:
        x (Tensor): The rows ``(T, K)``, sorted by group, float8_e4m3fn or float8_e5m2. ``K`` is a multiple of 16.
        scale_x (Tensor): float32 ``(T, ceil(K / 128))``, any strides.
        w (Tensor): One matrix per group ``(E, K, N)`` of either 8-bit type, ``N`` a multiple of 8, with ``K``
            contiguous (the order ``quantize_blocks`` returns); any other order is copied on every call.
        scale_w (Tensor): float32 ``(E, ceil(K / 128), ceil(N / 128))``, any strides.
        group_offsets (Tensor): As in :func:`grouped_matmul`.
        out_dtype (torch.dtype): float16, bfloat16 (default) or float32.

    Returns:
        Tensor: The products ``(T, N)``; rows of no group are zero.
    """
    if torch.compiler.is_compiling():
        if type(x) is not Tensor or type(w) not in _PLAIN or forward_mode() or (
                torch.is_grad_enabled() and (scale_x.requires_grad or scale_w.requires_grad or x.requires_grad
                                             or w.requires_grad)):
            return _grouped_matmul_scaled_no_compile(x, scale_x, w, scale_w, group_offsets, out_dtype)
        return _registered_scaled(x, scale_x, w, scale_w, group_offsets, out_dtype)
    impl = _grouped_matmul_scaled_eager if type(x) is Tensor and type(w) in _PLAIN else _grouped_matmul_scaled_plain
    return impl(x, scale_x, w, scale_w, group_offsets, out_dtype)
