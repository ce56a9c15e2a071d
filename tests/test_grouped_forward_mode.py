"""Forward-mode gradients of the grouped products and of the 8-bit rounding are refused, on the CPU: a dual tensor does
not require a gradient, and its tangent would be lost."""
import pytest
import torch
from torch.autograd import forward_ad

import blksprs_b200 as bs
from test_grouped_refusals import operands, scaled_operands


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("at", [0, 1])
def test_grouped_matmul_refuses_tangents(at):
    with forward_ad.dual_level():
        arguments = list(operands())
        with pytest.raises(ValueError, match="must be on GPU"):
            bs.ops.grouped_matmul(*arguments)
        arguments[at] = dual(arguments[at])
        with pytest.raises(ValueError, match="Forward-mode"):
            bs.ops.grouped_matmul(*arguments)
        with torch.no_grad(), pytest.raises(ValueError, match="Forward-mode"):
            bs.ops.grouped_matmul(*arguments)


@pytest.mark.parametrize("at", [1, 3])
def test_grouped_matmul_scaled_refuses_tangents(at):
    with forward_ad.dual_level():
        arguments = scaled_operands()
        with pytest.raises(ValueError, match="must be on GPU"):
            bs.ops.grouped_matmul_scaled(*arguments)
        arguments[at] = dual(arguments[at])
        with pytest.raises(ValueError, match="Forward-mode"):
            bs.ops.grouped_matmul_scaled(*arguments)


@pytest.mark.parametrize("op,shape", [(bs.ops.quantize_rows, (4, 40)), (bs.ops.quantize_blocks, (2, 4, 40))])
def test_quantize_refuses_tangents(op, shape):
    t = torch.zeros(shape)
    with forward_ad.dual_level():
        for value, message in ((t, "must be on GPU"), (dual(t), "Forward-mode")):
            with pytest.raises(ValueError, match=message):
                op(value)
