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


@pytest.mark.parametrize("out_dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("side", ["small", "large"])
@pytest.mark.parametrize("sizes,cols", [([1], 136), ([30, 0, 64, 1, 65], 136), ([5, 3], 4096), ([257, 1, 255, 0, 256], 392),
                                        ([600], 2056)], ids=str)
def test_scales_whose_product_leaves_fp32(sizes, cols, side, out_dtype):
    """Scales are any fp32 numbers: products of two below 2^-126 or above 2^128 next to ordinary ones, with sums that
    bring the result back into range, and sums of 0 where the product is infinite.  Both kernels of the product
    (few rows with and without a split contraction, many rows).  Multiplying twice is one rounding more than the one
    of the scales' product: the terms of a sum plus four, as for ordinary scales."""
    import blksprs_b200 as bs
    from test_gpu_p_grouped_matmul import assert_near, plain_scaled
    gen = torch.Generator().manual_seed(sum(sizes) + cols)
    rows, depth = sum(sizes), 1168
    blocks = -(-depth // 128)
    sign = -1.0 if side == "small" else 1.0
    # which rows have ordinary products, ones on either side of the border, and ones outside
    far = torch.tensor([0.0, 130.0, 142.0] if side == "small" else [0.0, 125.0, 130.0])
    far = far[torch.randint(0, 3, (rows, 1), generator=gen)]
    power = 70.0 + 5.0 * torch.randint(0, 3, (len(sizes), blocks, -(-cols // 128)), generator=gen)
    group = torch.repeat_interleave(torch.arange(len(sizes)), torch.tensor(sizes))

    def mantissa(*shape):
        return (1.0 + torch.rand(shape, generator=gen)) * (1 - 2 * torch.randint(0, 2, shape, generator=gen))
    # one exponent for a block of the rows whatever the columns: what a block of the weights has is taken off again
    sw = mantissa(*power.shape) * 2.0 ** (sign * power)
    sx = mantissa(rows, blocks) * 2.0 ** (sign * (far - 75.0))
    # values whose sums are large where the scales are small, and small where they are large
    magnitude = 2.0 ** (13 if side == "small" else -12)
    x = torch.randn((rows, depth), generator=gen) * magnitude
    x[torch.rand((rows, blocks), generator=gen).repeat_interleave(128, 1)[:, :depth] < 0.2] = 0.0
    w = torch.randn((len(sizes), cols, depth), generator=gen) * magnitude
    x, w = x.to(torch.float8_e5m2).to(DEV), w.to(torch.float8_e5m2).to(DEV).transpose(1, 2)
    sx, sw, offsets = sx.to(DEV), sw.to(DEV), bounds_of(sizes).to(DEV)
    products = sx.double()[:, :, None] * sw.double()[group.to(DEV)]
    outside = (products.abs() < 2.0 ** -126) | (products.abs() >= 2.0 ** 128)
    assert sx.isfinite().all() and sw.isfinite().all() and (rows < 8 or outside.any())
    want, magnitudes = plain_scaled(x, sx, w, sw, offsets)
    # no result overflows; the tolerance of the sums (2^-12.8 of their magnitude) covers half of bf16's smallest step, 2^-134
    assert magnitudes.max() < 2.0 ** 127 and magnitudes[magnitudes > 0].min() > 2.0 ** -121
    got = bs.ops.grouped_matmul_scaled(x, sx, w, sw, offsets, out_dtype=out_dtype)
    assert_near(got, want, magnitudes, depth + 4)


def test_scales_of_any_kind():
    """A scale of 0, infinity or NaN reaches its own rows and columns only, next to products out of range."""
    import blksprs_b200 as bs
    from test_gpu_p_grouped_matmul import make_scaled
    for sizes in ([40, 30], [400, 300]):
        x, sx, w, sw, offsets = make_scaled(sizes, 256, 264, seed=2)
        sx.fill_(2.0 ** -10)
        sw[:, :, 2] = 3e38
        clean = bs.ops.grouped_matmul_scaled(x, sx, w, sw, offsets)
        assert clean.isfinite().all()
        sx[3], sx[5, 1], sx[7, 0], sx[9], sx[11] = 0.0, float("nan"), float("inf"), 1e38, -1e-42
        out = bs.ops.grouped_matmul_scaled(x, sx, w, sw, offsets)
        assert not out[3].any() and out[5].isnan().all() and not out[7].isfinite().any()
        keep = torch.ones(x.shape[0], dtype=torch.bool, device=DEV)
        keep[[3, 5, 7, 9, 11]] = False
        assert torch.equal(out[keep], clean[keep])
        sw[1, 0, 1] = float("inf")
        other = bs.ops.grouped_matmul_scaled(x, sx, w, sw, offsets)
        assert not other[sizes[0]:, 128:256].isfinite().any()
        assert torch.equal(other[sizes[0]:, :128], clean[sizes[0]:, :128])
        assert torch.equal(other[sizes[0]:, 256:], clean[sizes[0]:, 256:])


@pytest.mark.parametrize("to", [torch.float8_e4m3fn, torch.float8_e5m2], ids=["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
def test_quantize_keeps_the_sign_of_zero(dtype, to):
    """Zeros of either sign, and values so small that they round to one, next to ordinary values and in a block of zeros."""
    import blksprs_b200 as bs
    from test_gpu_p_grouped_matmul import LARGEST, blocked, plain_quantize, plain_scale
    gen = torch.Generator().manual_seed(41)
    x = torch.randn((128, 384), generator=gen)
    x[torch.rand(x.shape, generator=gen) < 0.2] = 0.0
    x[torch.rand(x.shape, generator=gen) < 0.2] *= 2.0 ** -14
    x[:, 256:] = 0.0
    x = torch.where(torch.rand(x.shape, generator=gen) < 0.5, -x.abs(), x.abs()).to(dtype).to(DEV)
    q, scale = bs.ops.quantize_rows(x, to)
    want = plain_scale(x.float().reshape(128, 3, 128).abs().amax(2), to)
    assert torch.equal(scale, want)
    codes = q.view(torch.uint8)
    assert torch.equal(codes, plain_quantize(x, LARGEST[to], blocked(want, (1,)), to).view(torch.uint8))
    assert int((codes == 0x80).sum()) > 1000 and int((codes == 0).sum()) > 1000
    want = plain_scale(x.float().reshape(1, 128, 3, 128).abs().amax((1, 3)), to).reshape(1, 1, 3)
    codes = plain_quantize(x[None], LARGEST[to], blocked(want, (1, 2)), to)
    for w in (x[None], x.t().contiguous().t()[None]):
        q, scale = bs.ops.quantize_blocks(w, to)
        assert torch.equal(scale, want) and torch.equal(q.contiguous().view(torch.uint8), codes.view(torch.uint8))


def test_a_tangent_of_the_output_s_gradient_is_refused():
    import blksprs_b200 as bs
    from torch.autograd import forward_ad
    gen = torch.Generator().manual_seed(3)
    x, w, grad = whole(20, 32, gen=gen), whole(2, 32, 40, gen=gen), whole(20, 40, gen=gen)
    offsets = bounds_of([11, 9]).to(DEV)
    want = torch.autograd.grad(bs.ops.grouped_matmul(x.requires_grad_(True), w, offsets), x, grad)[0]
    with forward_ad.dual_level():
        assert torch.equal(torch.autograd.grad(bs.ops.grouped_matmul(x, w, offsets), x, grad)[0], want)
        out = bs.ops.grouped_matmul(x, w, offsets)
        with pytest.raises(ValueError, match="Forward-mode"):
            torch.autograd.grad(out, x, forward_ad.make_dual(grad, torch.ones_like(grad)))


def test_registered_operators():
    """Schemas, fake implementations and autograd of the operators a compiled caller calls."""
    import blksprs_b200  # noqa: F401
    ops = torch.ops.blksprs_b200
    gen = torch.Generator().manual_seed(4)
    x, w, grad, offsets = whole(20, 32, gen=gen), whole(2, 32, 40, gen=gen), whole(20, 40, gen=gen), bounds_of([11, 9]).to(DEV)
    f8 = torch.float8_e4m3fn
    wq, sw = ops.quantize_blocks(w, f8)
    xq, sx = ops.quantize_rows(x, f8)
    checks = ("test_schema", "test_autograd_registration", "test_faketensor")
    for stored in (w, w.transpose(1, 2).contiguous().transpose(1, 2)):
        torch.library.opcheck(ops.grouped_matmul.default, (x.clone().requires_grad_(), stored.clone().requires_grad_(), offsets),
                              test_utils=(*checks, "test_aot_dispatch_static"))
    torch.library.opcheck(ops.grouped_weight_gradient.default, (x, grad, offsets), test_utils=checks)
    checks = checks[1:]          # the schema's check multiplies what it is given and gets, which torch cannot in 8 bits
    torch.library.opcheck(ops.quantize_rows.default, (x, f8), test_utils=checks)
    torch.library.opcheck(ops.quantize_blocks.default, (w, f8), test_utils=checks)
    torch.library.opcheck(ops.grouped_matmul_scaled.default, (xq, sx, wq.transpose(1, 2), sw, offsets, BF16), test_utils=checks)


@pytest.mark.parametrize("stored", ["kn", "nk"])
def test_compiled_layer_of_experts_without_a_graph_break(stored):
    """Two products with an activation between, compiled whole: outputs and gradients of whole numbers equal the eager
    ones, for several numbers of rows, under autocast, and with a broadcast gradient."""
    import blksprs_b200 as bs
    gen = torch.Generator().manual_seed(5)
    up, down = whole(3, 32, 40, gen=gen), whole(3, 40, 24, gen=gen)
    if stored == "nk":
        up, down = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (up, down))

    def layer(x, up, down, offsets):
        hidden = torch.relu(bs.ops.grouped_matmul(x, up, offsets))
        return bs.ops.grouped_matmul(hidden * 2, down, offsets)

    compiled = torch.compile(layer, fullgraph=True)
    for rows in (16, 23, 300):
        x = whole(rows, 32, gen=gen)
        offsets = bounds_of([5, 0, rows - 7], 1).to(DEV)
        results = []
        for f in (compiled, layer):
            leaves = [t.clone().requires_grad_(True) for t in (x, up, down)]
            assert leaves[1].stride() == up.stride()
            out = f(*leaves, offsets)
            out.sum().backward()
            results.append([out.detach(), *(t.grad for t in leaves)])
        for got, want in zip(*results):
            assert got.dtype == want.dtype and torch.equal(got, want)
    with torch.autocast("cuda", dtype=BF16):
        args = (x.float(), up.float(), down.float(), offsets)
        got, want = compiled(*args), layer(*args)
    assert got.dtype == BF16 and torch.equal(got, want)


def test_compiled_serving_without_a_graph_break():
    import blksprs_b200 as bs
    from test_gpu_p_grouped_matmul import make
    x, w, _, offsets = make([10, 0, 61], 144, 136, BF16, seed=1, behind=3)

    def serve(x, wq, sw, offsets):
        xq, sx = bs.ops.quantize_rows(x)
        return bs.ops.grouped_matmul_scaled(xq, sx, wq, sw, offsets, out_dtype=FP32)

    def prepare(w):
        return bs.ops.quantize_blocks(w, torch.float8_e5m2)

    want_q, want_s = prepare(w)
    got_q, got_s = torch.compile(prepare, fullgraph=True)(w)
    assert got_q.stride() == want_q.stride() and torch.equal(got_s, want_s)
    assert torch.equal(got_q.transpose(1, 2).view(torch.uint8), want_q.transpose(1, 2).view(torch.uint8))
    compiled = torch.compile(serve, fullgraph=True)
    for part in (x, x[:40]):
        bounds = offsets.clamp(max=part.shape[0])
        assert torch.equal(compiled(part, want_q, want_s, bounds), serve(part, want_q, want_s, bounds))
    # what is refused without a compiler is refused with one
    for f, bad in ((lambda t: bs.ops.quantize_rows(t), x.float().requires_grad_(True)),
                   (lambda t: bs.ops.grouped_matmul(t, w, offsets), x[:, :136])):
        with pytest.raises(Exception, match="no gradient|Inner dimensions"):
            torch.compile(f)(bad)


def test_first_call_of_a_device_in_inference_mode(monkeypatch):
    """What it records is reported, and cleared, outside that mode."""
    import blksprs_b200 as bs
    from blksprs_b200 import _cabi, plan
    gen = torch.Generator().manual_seed(6)
    x, w = whole(20, 32, gen=gen), whole(2, 32, 40, gen=gen)
    monkeypatch.setattr(plan, "_status_words", {})
    with torch.inference_mode():
        bs.ops.grouped_matmul(x, w, bounds_of([11, 30]).to(DEV))
    with pytest.raises(_cabi.NativeError, match="range"):
        plan.check_device_status()
    plan.check_device_status()


def test_first_call_of_a_device_in_a_recording(monkeypatch):
    """Refused: the status word would lie in the graph's memory.  After a call outside it, replays neither clear nor lose
    what is recorded."""
    import blksprs_b200 as bs
    from blksprs_b200 import _cabi, plan
    gen = torch.Generator().manual_seed(6)
    x, w, offsets = whole(20, 32, gen=gen), whole(2, 32, 40, gen=gen), bounds_of([11, 9]).to(DEV)
    want = bs.ops.grouped_matmul(x, w, offsets)
    monkeypatch.setattr(plan, "_status_words", {})
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="once before recording"):
            bs.ops.grouped_matmul(x, w, offsets)
    bs.ops.grouped_matmul(x, w, offsets)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = bs.ops.grouped_matmul(x, w, offsets)
    bs.ops.grouped_matmul(x, w, bounds_of([11, 30]).to(DEV))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    with pytest.raises(_cabi.NativeError, match="range"):
        plan.check_device_status()
    graph.replay()
    plan.check_device_status()


def bad_bounds(good):
    """Bounds that decrease, start below 0, pass the rows' end, or hold anything; and what they are taken for."""
    rows, n = int(good[-1]), good.numel()
    low, high = torch.iinfo(good.dtype).min, torch.iinfo(good.dtype).max
    wild = good.clone()
    wild[::2] = torch.tensor([high, low, 7, -1, rows + 1])[torch.arange(wild[::2].numel()) % 5].to(good.dtype)
    swapped, below, beyond = good.flip(0), good.clone(), good.clone()
    if n > 3:
        swapped = good.clone()
        swapped[1], swapped[2] = good[2], good[1]
    below[0], beyond[-1] = -3, rows + 1
    for bad in (wild, swapped, below, beyond):
        yield bad, bad.long().clamp(0, rows).cummax(0).values.to(good.dtype)


@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["int32", "int64"])
@pytest.mark.parametrize("what,sizes,depth,cols", [
    ("few", [10, 20, 30], 64, 72), ("rows", [300, 257, 611, 1, 400], 136, 264), ("tall", [800] * 6, 72, 13320),
    ("gradient", [300, 257, 611, 1, 400], 136, 264), ("gradient", [500] * 8, 2048, 2568), ("gradient", [2500, 3000], 264, 136),
    ("gradient", [9000], 72, 72), ("scaled", [300, 257, 611, 1, 400], 144, 264), ("scaled", [10, 20, 30], 1040, 72)],
    ids=str)
def test_bad_bounds_in_every_kernel(what, sizes, depth, cols, index):
    """Clamped on the device before use, reported, and computed as the bounds they are taken for."""
    import blksprs_b200 as bs
    from blksprs_b200 import _cabi
    from blksprs_b200.plan import check_device_status
    gen = torch.Generator().manual_seed(depth)
    good, rows = bounds_of(sizes, dtype=index), sum(sizes)
    x = whole(rows, depth, gen=gen)
    if what == "gradient":
        grad = whole(rows, cols, gen=gen)

        def call(offsets):
            return weight_gradient(x, grad, offsets)
    elif what == "scaled":
        w = whole(len(sizes), cols, depth, gen=gen).to(torch.float8_e4m3fn).transpose(1, 2)
        sx = torch.ones((rows, -(-depth // 128)), device=DEV)
        sw = torch.ones((len(sizes), sx.shape[1], -(-cols // 128)), device=DEV)

        def call(offsets):
            return bs.ops.grouped_matmul_scaled(x.to(torch.float8_e4m3fn), sx, w, sw, offsets)
    else:
        w = whole(len(sizes), depth, cols, gen=gen)

        def call(offsets):
            return bs.ops.grouped_matmul(x, w, offsets)
    call(good.to(DEV))
    check_device_status()
    for bad, taken in bad_bounds(good):
        got = call(bad.to(DEV))
        with pytest.raises(_cabi.NativeError, match="range"):
            check_device_status()
        assert torch.equal(got, call(taken.to(DEV)))
        check_device_status()


@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("sizes,depth,cols", [([300, 257, 611, 1, 400], 136, 264), ([800, 513, 385, 1, 900, 640], 200, 13320)],
                         ids=["256", "tall"])
def test_values_that_are_not_finite_stay_in_their_row_of_many(sizes, depth, cols, stored):
    """The kernels of many rows: a NaN or infinity reaches its own row of the product and of the row gradient only; one in
    the weights its own group's."""
    import blksprs_b200 as bs
    gen = torch.Generator().manual_seed(cols)
    rows, at = sum(sizes) + 70, [0, 299, 300, 556, 900, sum(sizes) - 1, sum(sizes) + 3]
    x, grad = whole(rows, depth, gen=gen), whole(rows, cols, gen=gen)
    w = whole(len(sizes), depth, cols, gen=gen)
    w = w if stored == "kn" else w.transpose(1, 2).contiguous().transpose(1, 2)
    offsets = bounds_of(sizes).to(DEV)
    keep = torch.ones(rows, dtype=torch.bool, device=DEV)
    keep[at] = False

    def both(x, w, grad):
        x = x.detach().requires_grad_(True)
        out = bs.ops.grouped_matmul(x, w, offsets)
        return out.detach(), torch.autograd.grad(out, x, grad)[0]

    clean = both(x, w, grad)
    want = torch.cat([x[a:b].double() @ w[e].double() for e, (a, b) in enumerate(zip(offsets.tolist(), offsets[1:].tolist()))])
    assert torch.equal(clean[0][:sum(sizes)].double(), want) and not clean[0][sum(sizes):].any()
    x[at, 5], grad[at, 7] = float("nan"), float("inf")
    for got, wanted in zip(both(x, w, grad), clean):
        assert torch.equal(got[keep], wanted[keep])
        assert not got[at[:-1]].isfinite().all(1).any() and not got[at[-1]].any()
    x, grad = x.nan_to_num(0.0), grad.nan_to_num(0.0, 0.0)
    wanted = both(x, w, grad)
    w[1, 3, 4] = float("nan")
    group = slice(int(offsets[1]), int(offsets[2]))
    for got, want, column in zip(both(x, w, grad), wanted, (4, 3)):
        assert got[group, column].isnan().all()
        got[group, column] = want[group, column]
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [FP16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("sizes,depth,cols", [([40000], 128, 264), ([5, 20011, 0, 19990], 72, 136), ([3001] * 8, 520, 2056),
                                              ([9001, 7030], 2048, 4104)], ids=str)
def test_every_row_of_a_long_group_counts(sizes, depth, cols, dtype):
    """Weight gradients of long groups whose rows are zero but for a few at the ends of groups, of parts, of steps and of
    the last sixteen: sums small enough for the output type to hold, so that a row lost or counted twice shows."""
    gen = torch.Generator().manual_seed(depth + cols)
    rows = sum(sizes) + 24
    offsets = bounds_of(sizes, 8)
    x, grad = torch.zeros((rows, depth), dtype=dtype, device=DEV), torch.zeros((rows, cols), dtype=dtype, device=DEV)
    for a, b in zip(offsets.tolist(), offsets[1:].tolist()):
        steps = torch.randint(0, max(1, (b - a) // 64), (8,), generator=gen) * 64 + a
        ends = [range(a, a + 17), range(b - 66, b), *(range(s - 1, s + 2) for s in steps.tolist())]
        at = sorted({r for part in ends for r in part if a <= r < b})
        assert len(at) < 128
        x[at], grad[at] = whole(len(at), depth, gen=gen, dtype=dtype), whole(len(at), cols, gen=gen, dtype=dtype)
    x[:8], grad[:8], x[-16:], grad[-16:] = 1.0, 1.0, 1.0, 1.0          # rows of no group
    want = plain_weight_gradient(x, grad, offsets)
    assert want.abs().max() <= 256
    assert torch.equal(weight_gradient(x, grad, offsets.to(DEV)).double(), want)


@pytest.mark.parametrize("sizes,depth,cols", [([5, 0, 3], 4096, 136), ([1200, 1], 2056, 264), ([3000, 2500], 4104, 2568)], ids=str)
def test_every_value_of_a_long_contraction_counts(sizes, depth, cols):
    """The same of the rows product: values at the ends of its contraction, of steps and of a cluster's shares."""
    import blksprs_b200 as bs
    gen = torch.Generator().manual_seed(depth)
    x, w = whole(sum(sizes), depth, gen=gen, dtype=BF16), whole(len(sizes), depth, cols, gen=gen, dtype=BF16)
    keep = torch.zeros(depth, dtype=torch.bool)
    for s in [0, depth, depth // 2, *(torch.randint(1, depth // 64, (12,), generator=gen) * 64).tolist()]:
        keep[max(0, s - 4):s + 4] = True
    x[:, ~keep.to(DEV)] = 0
    offsets = bounds_of(sizes)
    want = torch.cat([x[a:b].double() @ w[e].double() for e, (a, b) in enumerate(zip(offsets.tolist(), offsets[1:].tolist()))])
    assert want.abs().max() <= 256
    for stored in (w, w.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(bs.ops.grouped_matmul(x, stored, offsets.to(DEV)).double(), want)


def test_registered_weight_gradient_refuses_what_would_be_read_out_of_bounds():
    import blksprs_b200  # noqa: F401
    op = torch.ops.blksprs_b200.grouped_weight_gradient
    x, grad, offsets = (torch.zeros(s, dtype=BF16, device=DEV) for s in ((20, 32), (20, 40), (3,)))
    offsets = offsets.int()
    assert op(x, grad, offsets).shape == (2, 32, 40)
    for bad, message in (((x, grad[:10], offsets), "rows"), ((x[0], grad, offsets), "2 dimensions"),
                         ((x, grad.half(), offsets), "same dtype"), ((x.float(), grad.float(), offsets), "float16 or"),
                         ((x, grad[:, :36], offsets), "divisible"), ((x[:, :28], grad, offsets), "divisible"),
                         ((x, grad, offsets.float()), "int32 or int64"), ((x, grad, offsets[:0]), "one entry more"),
                         ((x, grad, offsets[None]), "one entry more"), ((x, grad, offsets.repeat(2)[::2]), "contiguous"),
                         ((x, grad, offsets.cpu()), "same device"), ((x, grad, offsets.repeat(342)), "at most 1024")):
        with pytest.raises(ValueError, match=message):
            op(*bad)


def test_tangents_of_registered_and_compiled_calls_are_refused():
    import blksprs_b200 as bs
    from torch.autograd import forward_ad
    gen = torch.Generator().manual_seed(3)
    x, w, offsets = whole(20, 32, gen=gen), whole(2, 32, 40, gen=gen), bounds_of([11, 9]).to(DEV)
    wq, sw = bs.ops.quantize_blocks(w)
    xq, sx = bs.ops.quantize_rows(x)
    ops = torch.ops.blksprs_b200
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        ds = forward_ad.make_dual(sx, torch.ones_like(sx))
        for f in (lambda: ops.grouped_matmul(d, w, offsets), lambda: ops.grouped_weight_gradient(x, d, offsets),
                  lambda: ops.quantize_rows(d, torch.float8_e4m3fn),
                  lambda: ops.grouped_matmul_scaled(xq, ds, wq, sw, offsets, BF16),
                  lambda: torch.compile(lambda t: bs.ops.grouped_matmul(t, w, offsets), backend="eager")(d),
                  lambda: torch.compile(lambda t: bs.ops.quantize_rows(t), backend="eager")(d)):
            with pytest.raises(ValueError, match="Forward-mode"):
                f()
