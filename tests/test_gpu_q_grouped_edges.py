"""Grouped products and 8-bit rounding where they can go wrong at their edges: both kernels of each product, values that
are not finite next to a group, very wide outputs, scales far from one, recorded and forward-mode calls.

Most operands are small whole numbers, so that every product and sum is exact in the output type and results have to be
equal; the other tolerances are those of the grouped products' own tests.
"""
import pytest
import torch

from gpu_util import DEV
from test_gpu_p_grouped_matmul import BF16, FP16, FP32, bounds_of, plain_weight_gradient

pytestmark = pytest.mark.gpu


def whole(*shape, gen, dtype=FP16, high=1):
    return torch.randint(-high, high + 1, shape, generator=gen).to(dtype).to(DEV)


def weight_gradient(x, grad, offsets):
    import blksprs_b200 as bs
    w = torch.zeros((offsets.numel() - 1, x.shape[1], grad.shape[1]), dtype=x.dtype, device=DEV).requires_grad_(True)
    return torch.autograd.grad(bs.ops.grouped_matmul(x, w, offsets), w, grad)[0]


# sizes of groups, depth, columns: tiles of 256 rows, of 512 rows (a few hundred tiles, long groups), rows in parts
GRADIENT_FORMS = [([17, 1, 31, 63, 79, 95, 15, 130], 264, 392), ([33] * 40, 136, 520),
                  ([385 + 13 * i for i in range(8)], 2048, 2568), ([4101], 264, 136), ([3, 9000, 2], 72, 264)]


@pytest.mark.parametrize("sizes,depth,cols", GRADIENT_FORMS, ids=["short", "equal", "tall", "parts", "parts-of-one"])
def test_weight_gradient_keeps_out_the_rows_of_other_groups(sizes, depth, cols):
    """The last rows of a group share sixteen rows of a tile with the next group's, which are NaN and infinity here in
    every second group and behind the last; both blocks of a pair clear theirs before one of them multiplies."""
    gen = torch.Generator().manual_seed(depth)
    before, behind = 5, 40
    rows = before + sum(sizes) + behind
    x, grad, offsets = whole(rows, depth, gen=gen), whole(rows, cols, gen=gen), bounds_of(sizes, before).to(DEV)
    want = plain_weight_gradient(x, grad, offsets)
    assert want.abs().max() <= 2048        # whole numbers that fp16 holds
    bounds = offsets.tolist()
    for clean in (0, 1):
        spoilt, spoilt_grad = x.clone(), grad.clone()
        for e, (a, b) in enumerate(zip([0, *bounds], [*bounds, rows])):      # part e is group e - 1
            if e % 2 != clean or e in (0, len(bounds)):
                spoilt[a:b], spoilt_grad[a:b] = float("nan"), float("inf")
        for _ in range(3):
            got = weight_gradient(spoilt, spoilt_grad, offsets)
            for e in range(len(sizes)):
                if (e + 1) % 2 == clean:
                    assert torch.equal(got[e].double(), want[e]), (clean, e)


def test_parts_are_joined_after_they_are_written():
    """Many split weight gradients one behind the other, every one on other rows and in the workspace of the one before."""
    gen = torch.Generator().manual_seed(31)
    offsets = bounds_of([8200]).to(DEV)
    x, grad = whole(8200, 64, gen=gen), whole(8200, 136, gen=gen)
    got = [weight_gradient(x.roll(i, 0), grad, offsets) for i in range(60)]
    for i, g in enumerate(got):
        want = plain_weight_gradient(x.roll(i, 0), grad, offsets)
        assert want.abs().max() <= 2048 and torch.equal(g.double(), want), i


def spoil_free_memory(*shape):
    """What the next allocation of this size holds before it is written."""
    torch.empty(shape, dtype=torch.int16, device=DEV).fill_(-1)


def test_more_than_2_to_30_columns():
    """Byte counts behind a column pass 31 bits: the forward product of one row and the weight gradient of two."""
    import blksprs_b200 as bs
    cols = 2 ** 30 + 8
    gen = torch.Generator().manual_seed(7)
    x = torch.zeros((1, 8), dtype=BF16, device=DEV)
    x[0, 3] = 2.0
    w = torch.empty((1, 8, cols), dtype=BF16, device=DEV)
    line = whole(2 ** 20, gen=gen, dtype=BF16, high=9)
    for k in range(8):
        w[0, k, :2 ** 30].view(-1, 2 ** 20).copy_(line.roll(k))
        w[0, k, 2 ** 30:] = k + 1
    offsets = bounds_of([1]).to(DEV)
    spoil_free_memory(1, cols)
    out = bs.ops.grouped_matmul(x, w, offsets)
    assert torch.equal(out, 2 * w[0, 3:4])
    grad = w[0, 2:4].clone()
    del out, w
    torch.cuda.empty_cache()
    x = whole(2, 8, gen=gen, dtype=BF16, high=3)
    w = torch.empty((1, 8, cols), dtype=BF16, device=DEV).requires_grad_(True)
    product = bs.ops.grouped_matmul(x, w, bounds_of([2]).to(DEV))
    spoil_free_memory(1, 8, cols)
    got, = torch.autograd.grad(product, w, grad)
    for k in range(8):
        assert torch.equal(got[0, k], x[0, k] * grad[0] + x[1, k] * grad[1]), k
    del got, w, grad, product
    torch.cuda.empty_cache()


def test_nearly_2_to_31_rows():
    """Heights of tiles are found without leaving 31 bits: one group of 2^31 - 520 rows, and a weight gradient of as many."""
    import sys
    import blksprs_b200 as bs
    rows, part = 2 ** 31 - 520, 2 ** 20
    gen = torch.Generator().manual_seed(8)
    line, w = whole(part, 8, gen=gen, dtype=BF16, high=3), whole(1, 8, 8, gen=gen, dtype=BF16, high=3)
    times, rest = divmod(rows, part)
    x = torch.empty((rows, 8), dtype=BF16, device=DEV)
    x[:times * part].view(times, part, 8).copy_(line)
    x[times * part:] = line[:rest]
    spoil_free_memory(rows, 8)
    out = bs.ops.grouped_matmul(x, w, torch.tensor([0, rows], device=DEV))
    want = (line.double() @ w[0].double()).to(BF16)
    for i in range(0, times, 64):
        assert bool((out[i * part:min(i + 64, times) * part].view(-1, part, 8) == want).all()), i
    assert torch.equal(out[times * part:], want[:rest])
    del out, x
    torch.cuda.empty_cache()
    x = torch.empty((2, rows), dtype=BF16, device=DEV)
    for r in range(2):
        x[r, :times * part].view(times, part).copy_(line[:, r])
        x[r, times * part:] = r + 1
    grad = whole(2, 8, gen=gen, dtype=BF16, high=3)
    spoil_free_memory(1, rows, 8)
    got = sys.modules["blksprs_b200.ops.grouped_matmul"]._weight_gradient(x, grad, bounds_of([2]).to(DEV), 1)
    for c in range(8):
        assert torch.equal(got[0, :, c], x[0] * grad[0, c] + x[1] * grad[1, c]), c
    del got, x, grad
    torch.cuda.empty_cache()
