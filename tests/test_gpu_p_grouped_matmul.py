"""Products grouped by expert and 8-bit rounding with block scales against plain forms in 64 bits.

Tolerances.  A product of 16-bit operands is exact in fp32 up to its own rounding, so what an output may be off by is
the sum's error and the last rounding: with A = |x| @ |w| a sum of n terms held in fp32, each addition truncated at
worst, is off by at most n * 2^-23 * A, and rounding to the output type by at most half a step of the value
(eps / 2 relative; for fp16 at least half its smallest step, 2^-25).  The scaled product adds two roundings of its
factors: (n + 4) * 2^-23.
"""
import pytest
import torch

from gpu_util import DEV

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
LARGEST = {E4M3: 448.0, E5M2: 57344.0}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_near(got, want, magnitudes, terms, what=""):
    """``got`` against 64-bit ``want``; ``magnitudes`` = the same sum of absolute values."""
    assert got.shape == want.shape
    want, magnitudes = want.to(got.device), magnitudes.to(got.device)
    allowed = terms * 2.0 ** -23 * magnitudes
    allowed = allowed + half_step(got.dtype) * (want.abs() + allowed) + (2.0 ** -25 if got.dtype == FP16 else 0.0)
    off = (got.double() - want).abs() - allowed
    assert not torch.isnan(got.double()).any(), what
    assert off.numel() == 0 or float(off.max()) <= 0.0, (what, float(off.max()), int((off > 0).sum()))


def bounds_of(sizes, first=0, dtype=torch.int32):
    offsets = torch.zeros(len(sizes) + 1, dtype=torch.int64)
    offsets[1:] = torch.cumsum(torch.tensor(sizes, dtype=torch.int64), 0)
    return (offsets + first).to(dtype)


def plain(x, w, offsets):
    """Rows product in 64 bits on the operands' device."""
    out = torch.zeros((x.shape[0], w.shape[2]), dtype=torch.float64, device=x.device)
    bounds = offsets.tolist()
    for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
        out[a:b] = x[a:b].double() @ w[e].double()
    return out


def plain_weight_gradient(x, grad, offsets):
    bounds = offsets.tolist()
    return torch.stack([x[a:b].double().t() @ grad[a:b].double() for a, b in zip(bounds, bounds[1:])])


def values(*shape, dtype, gen, scale=1.0):
    return (torch.randn(shape, generator=gen) * scale).to(dtype).to(DEV)


def make(sizes, depth, cols, dtype, seed=0, before=0, behind=0, stored="kn", index=torch.int32):
    gen = torch.Generator().manual_seed(seed)
    rows = before + sum(sizes) + behind
    x = values(rows, depth, dtype=dtype, gen=gen)
    if stored == "kn":
        w = values(len(sizes), depth, cols, dtype=dtype, gen=gen, scale=depth ** -0.5)
    else:
        w = values(len(sizes), cols, depth, dtype=dtype, gen=gen, scale=depth ** -0.5).transpose(1, 2)
    grad = values(rows, cols, dtype=dtype, gen=gen)
    return x, w, grad, bounds_of(sizes, before, index).to(DEV)


def check_training(x, w, grad, offsets):
    import blksprs_b200 as bs
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    out = bs.ops.grouped_matmul(x, w, offsets)
    grad_x, grad_w = torch.autograd.grad(out, (x, w), grad)
    x, w, out = x.detach(), w.detach(), out.detach()
    assert out.dtype == grad_x.dtype == grad_w.dtype == x.dtype
    assert_near(out, plain(x, w, offsets), plain(x.abs(), w.abs(), offsets), x.shape[1], "out")
    wt = w.transpose(1, 2)
    assert_near(grad_x, plain(grad, wt, offsets), plain(grad.abs(), wt.abs(), offsets), w.shape[2], "grad_x")
    longest = int((offsets[1:] - offsets[:-1]).max())
    assert_near(grad_w, plain_weight_gradient(x, grad, offsets),
                plain_weight_gradient(x.abs(), grad.abs(), offsets), max(longest, 1), "grad_w")
    from blksprs_b200.plan import check_device_status
    check_device_status()


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("sizes", [
    [1], [16], [31, 0, 33], [0, 0, 5], [257, 1, 255, 0, 256], [15, 17, 64, 63, 65, 129], [700],
], ids=str)
def test_sizes_of_groups(sizes, stored, dtype):
    check_training(*make(sizes, 72, 136, dtype, seed=len(sizes), stored=stored))


@pytest.mark.parametrize("depth,cols", [(8, 8), (64, 128), (128, 64), (200, 264), (520, 24), (24, 520), (1032, 392)])
def test_odd_depths_and_columns(depth, cols):
    check_training(*make([37, 0, 300], depth, cols, BF16, seed=depth))
    check_training(*make([37, 0, 300], depth, cols, FP16, seed=cols, stored="nk"))


@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("sizes", [[4097, 4999], [8191, 1, 0, 800], [9729]], ids=str)
def test_long_groups(sizes, stored):
    """Enough tiles for the tall ones (up to 512 rows), heights that do not divide."""
    check_training(*make(sizes, 72, 4104, BF16, seed=len(sizes), stored=stored, before=3, behind=30))


@pytest.mark.parametrize("stored", ["kn", "nk"])
def test_weight_gradient_of_large_weights(stored):
    """Tall tiles of the weight gradient: contractions whose last rows are and are not a multiple of 16."""
    check_training(*make([403, 512, 0, 700, 385, 416], 2056, 4104, FP16, seed=11, stored=stored, behind=5))


@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("depth,cols", [(512, 136), (1032, 200), (2048, 128), (4160, 72)])
@pytest.mark.parametrize("sizes", [[1], [0, 2, 0, 1], [30, 0, 64, 1, 65], [0] * 40 + [33]], ids=str)
def test_few_rows_split_over_the_depth(sizes, depth, cols, stored):
    """Few tiles and a long contraction: the sums of a tile are split over two to eight thread blocks."""
    check_training(*make(sizes, depth, cols, BF16, seed=depth, stored=stored, before=1, behind=2))


@pytest.mark.parametrize("out_dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("depth,cols", [(1024, 136), (2064, 200), (4096, 128), (8320, 72)])
@pytest.mark.parametrize("sizes", [[1], [0, 2, 0, 1], [30, 0, 64, 1, 65], [0] * 40 + [33]], ids=str)
def test_scaled_few_rows_split_over_the_depth(sizes, depth, cols, out_dtype):
    check_scaled(*make_scaled(sizes, depth, cols, seed=depth, before=1, behind=2), out_dtype)


@pytest.mark.parametrize("before,behind", [(0, 7), (5, 0), (130, 300), (1, 1)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["int32", "int64"])
def test_rows_of_no_group_are_zero(before, behind, index):
    check_training(*make([3, 0, 129, 40], 64, 72, BF16, seed=before, before=before, behind=behind, index=index))


def test_all_groups_empty():
    import blksprs_b200 as bs
    x, w, grad, offsets = make([0, 0, 0], 64, 72, BF16, behind=9)
    check_training(x, w, grad, offsets)
    assert not bs.ops.grouped_matmul(x, w, offsets).any()


def test_no_rows_no_groups():
    import blksprs_b200 as bs
    x, w, grad, offsets = make([0, 0], 64, 72, BF16)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    out = bs.ops.grouped_matmul(x, w, offsets)
    assert out.shape == (0, 72)
    grad_x, grad_w = torch.autograd.grad(out, (x, w), grad)
    assert grad_x.shape == x.shape and grad_w.shape == w.shape and not grad_w.any()
    out = bs.ops.grouped_matmul(torch.ones((3, 64), dtype=BF16, device=DEV), w.detach()[:0],
                                torch.zeros(1, dtype=torch.int32, device=DEV))
    assert out.shape == (3, 72) and not out.any()


def test_many_groups():
    gen = torch.Generator().manual_seed(3)
    sizes = torch.randint(0, 6, (1024,), generator=gen).tolist()
    check_training(*make(sizes, 64, 72, BF16, seed=4))


def test_values_that_are_not_finite_stay_in_their_row():
    """A NaN or infinity in one row reaches that row's output only, and in the gradient its own group's only; rows
    behind the last group reach nothing."""
    import blksprs_b200 as bs
    x, w, grad, offsets = make([20, 21, 22], 64, 72, BF16, seed=8, behind=6)
    clean = bs.ops.grouped_matmul(x, w, offsets)
    clean_w = torch.autograd.grad(bs.ops.grouped_matmul(x, w.requires_grad_(True), offsets), w, grad)[0]
    w = w.detach()
    spoilt, spoilt_grad = x.clone(), grad.clone()
    spoilt[20, 3], spoilt[-1], spoilt_grad[-2] = float("nan"), float("inf"), float("nan")
    out = bs.ops.grouped_matmul(spoilt, w, offsets)
    assert out[20].isnan().all()
    keep = torch.arange(x.shape[0], device=DEV) != 20
    assert torch.equal(out[keep], clean[keep])
    grad_w = torch.autograd.grad(bs.ops.grouped_matmul(spoilt, w.requires_grad_(True), offsets), w, spoilt_grad)[0]
    assert torch.equal(grad_w[[0, 2]], clean_w[[0, 2]])
    assert grad_w[1, 3].isnan().all() and torch.equal(grad_w[1, 4:], clean_w[1, 4:])


def test_strided_and_unaligned_operands():
    import blksprs_b200 as bs
    gen = torch.Generator().manual_seed(5)
    offsets = bounds_of([40, 3, 90]).to(DEV)
    wide = values(133, 3 * 64 + 8, dtype=BF16, gen=gen)
    weights = values(3, 64, 80, dtype=BF16, gen=gen)
    for x in (wide[:, 64:128], wide[:, 3:67], wide.t().contiguous().t()[:, :64], wide[:1].expand(133, -1)[:, :64]):
        for w in (weights, weights[:, :, 8:80], weights[:, :, 4:76], weights.flip(0)[:, :, :72],
                  weights[:1].expand(3, -1, -1)):
            check_training(x, w, values(133, w.shape[2], dtype=BF16, gen=gen), offsets)
    x, w = wide[:, :64], weights
    grad = values(1, 80, dtype=BF16, gen=gen).expand(133, -1)
    check_training(x, w, grad, offsets)
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    bs.ops.grouped_matmul(x, w, offsets).sum().backward()          # a gradient that is one broadcast value
    assert_near(w.grad, plain_weight_gradient(x.detach(), torch.ones_like(grad), offsets),
                plain_weight_gradient(x.detach().abs(), torch.ones_like(grad), offsets), 90)


def test_gradients_against_differences():
    """The directional difference of a quadratic loss, on values whose products and sums are exact in fp16."""
    import blksprs_b200 as bs
    gen = torch.Generator().manual_seed(6)
    offsets = bounds_of([5, 0, 11]).to(DEV)

    def small(*shape):
        return torch.randint(-2, 3, shape, generator=gen).to(FP16).to(DEV)

    x, w, dx, dw, g = small(16, 32), small(3, 32, 40), small(16, 32), small(3, 32, 40), small(16, 40)
    x.requires_grad_(True), w.requires_grad_(True)
    grad_x, grad_w = torch.autograd.grad(bs.ops.grouped_matmul(x, w, offsets), (x, w), g)
    with torch.no_grad():
        def loss(a, b):
            return (bs.ops.grouped_matmul(a, b, offsets).double() * g.double()).sum()
        # the product is bilinear: the central difference along one argument is exact
        along_x = (loss(x + dx, w) - loss(x - dx, w)) / 2
        along_w = (loss(x, w + dw) - loss(x, w - dw)) / 2
    assert float(along_x) == float((grad_x.double() * dx.double()).sum())
    assert float(along_w) == float((grad_w.double() * dw.double()).sum())


def test_bad_bounds_are_clamped_and_reported():
    """Offsets that decrease or leave the rows: every access stays in bounds (they are clamped before use, which the
    kernel does for all of them alike), the status word tells, and later calls are not affected."""
    import blksprs_b200 as bs
    from blksprs_b200 import _cabi
    from blksprs_b200.plan import check_device_status
    x, w, grad, offsets = make([10, 20, 30], 64, 72, BF16)
    for bad in ([0, 10, 5, 60], [-3, 10, 30, 60], [0, 10, 30, 61], [0, 2 ** 31 - 1, -2 ** 31, 7]):
        bs.ops.grouped_matmul(x, w, torch.tensor(bad, dtype=torch.int32, device=DEV))
        with pytest.raises(_cabi.NativeError, match="range"):
            check_device_status()
    bs.ops.grouped_matmul(x, w, torch.tensor([0, 10, 30, 2 ** 40], device=DEV))
    with pytest.raises(_cabi.NativeError, match="range"):
        check_device_status()
    check_training(x, w, grad, offsets)


def test_other_stream_and_graph_replay():
    import blksprs_b200 as bs
    x, w, grad, offsets = make([10, 300, 0, 77], 64, 136, BF16, behind=5)
    want = bs.ops.grouped_matmul(x, w, offsets)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = bs.ops.grouped_matmul(x, w, offsets)
        q, s = bs.ops.quantize_rows(x)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            recorded = bs.ops.grouped_matmul(x, w, offsets)
            rq, rs = bs.ops.quantize_rows(x)
    assert torch.equal(got, want)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(recorded, want) and torch.equal(rq.view(torch.uint8), q.view(torch.uint8)) and torch.equal(rs, s)
    # other bounds and rows in the same buffers
    x.copy_(x.flip(0))
    offsets.copy_(bounds_of([200, 1, 100, 80], 3).to(DEV))
    graph.replay()
    torch.cuda.synchronize()
    replayed = recorded.clone()
    assert torch.equal(replayed, bs.ops.grouped_matmul(x, w, offsets))
    assert not torch.equal(replayed, want)


def test_recorded_training_step_and_serving_call():
    """A training step (gradients of leaves that no eager graph holds) and a serving call, recorded and replayed on
    other values, bounds and scales in the same buffers."""
    import blksprs_b200 as bs
    x, w, grad, offsets = make([10, 300, 0, 77], 144, 136, BF16, behind=5)

    def training(a, b):
        out = bs.ops.grouped_matmul(a, b, offsets)
        return (out.detach(), *torch.autograd.grad(out, (a, b), grad))

    def serving():
        xq, sx = bs.ops.quantize_rows(x)
        wq, sw = bs.ops.quantize_blocks(w)
        return (bs.ops.grouped_matmul_scaled(xq, sx, wq, sw, offsets), sx, sw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        training(x.detach().requires_grad_(True), w.detach().requires_grad_(True))
        serving()
        side.synchronize()
        leaves = [t.detach().requires_grad_(True) for t in (x, w)]
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            recorded = (*training(*leaves), *serving())
    for shift in (0, 1):
        if shift:
            x.copy_(x.flip(0)), w.copy_(w.flip(0)), grad.copy_(grad.flip(1))
            offsets.copy_(bounds_of([200, 1, 100, 80], 3).to(DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in recorded]
        want = (*training(x.detach().requires_grad_(True), w.detach().requires_grad_(True)), *serving())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_backward_copies_whatever_the_switch_for_inputs_says():
    import blksprs_b200 as bs
    x, w, grad, offsets = make([10, 30], 64, 72, BF16)
    bs.utils.disable_contiguous()
    try:
        with pytest.raises(ValueError, match="contiguous"):
            bs.ops.grouped_matmul(x[:, 4:60], w[:, 4:60], offsets)
        w.requires_grad_(True)
        out = bs.ops.grouped_matmul(x, w, offsets)
        got, = torch.autograd.grad(out, w, grad[:, :1].expand(-1, 72))
    finally:
        bs.utils.enable_contiguous()
    want, = torch.autograd.grad(bs.ops.grouped_matmul(x, w, offsets), w, grad[:, :1].repeat(1, 72))
    assert torch.equal(got, want)


def test_two_streams_at_once():
    import blksprs_b200 as bs
    cases = [make([10, 300, 0, 77], 520, 1032, BF16, seed=1), make([2, 0, 1, 3], 2048, 512, FP16, seed=2, stored="nk"),
             make([2000, 1, 999], 264, 520, BF16, seed=3, behind=9)]
    for x, w, _, _ in cases:
        x.requires_grad_(True), w.requires_grad_(True)

    def step(x, w, grad, offsets):
        out = bs.ops.grouped_matmul(x, w, offsets)
        return (out.detach(), *torch.autograd.grad(out, (x, w), grad))
    want = [step(*case) for case in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(5):
        for stream, case, results in zip(streams, cases, got):
            with torch.cuda.stream(stream):
                results.append(step(*case))
    torch.cuda.synchronize()
    for results, wanted in zip(got, want):
        for result in results:
            assert all(torch.equal(a, b) for a, b in zip(result, wanted))


def test_output_beyond_32_bit_offsets():
    """2.3e9 output elements: the last rows and columns, from both ends of the offsets."""
    import blksprs_b200 as bs
    gen = torch.Generator().manual_seed(12)
    rows, cols = 70001, 32776
    x, w = values(rows, 64, dtype=BF16, gen=gen), values(2, 64, cols, dtype=BF16, gen=gen, scale=0.125)
    offsets = bounds_of([69990, 9], 1).to(DEV)
    out = bs.ops.grouped_matmul(x, w, offsets)
    for part, e in ((slice(1, 9), 0), (slice(65530, 65545), 0), (slice(69985, 69991), 0), (slice(69991, 70000), 1)):
        assert_near(out[part], x[part].double() @ w[e].double(), x[part].double().abs() @ w[e].double().abs(), 64)
    assert not out[0].any() and not out[70000].any()


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("stored", ["kn", "nk"])
@pytest.mark.parametrize("sizes,depth,cols", [
    ([1024], 8, 8), ([4100], 264, 136), ([1, 0, 12345, 70, 3], 72, 264), ([0, 9000, 0], 520, 40), ([5000, 5001], 256, 512),
    ([40000], 128, 1032)], ids=str)
def test_weight_gradient_in_parts(sizes, depth, cols, stored, dtype):
    """Few tiles, many rows: parts without rows, parts that end inside a step, rows before and behind the groups."""
    from blksprs_b200 import _cabi
    x, w, grad, offsets = make(sizes, depth, cols, dtype, seed=depth, stored=stored, before=9, behind=21)
    assert _cabi.lib().bsp_grouped_weight_grad_workspace(x.shape[0], len(sizes), depth, cols) > 0
    x[:9] = grad[-21:] = float("nan")
    check_training(torch.nan_to_num(x), w, torch.nan_to_num(grad), offsets)
    import blksprs_b200 as bs
    x, w = x.requires_grad_(), w.requires_grad_()
    first = torch.autograd.grad(bs.ops.grouped_matmul(x, w, offsets), w, grad)[0]
    clean = torch.autograd.grad(bs.ops.grouped_matmul(torch.nan_to_num(x.detach()), w, offsets), w, torch.nan_to_num(grad))[0]
    assert torch.equal(first, clean)


def test_weight_gradient_needs_its_workspace():
    """Refused before anything is launched: no workspace, one that is too small, one that is not aligned."""
    from blksprs_b200 import _cabi
    x, w, grad, offsets = make([5000], 64, 72, BF16)
    lib, out = _cabi.lib(), torch.full((1, 64, 72), 3.0, dtype=BF16, device=DEV)
    size = lib.bsp_grouped_weight_grad_workspace(5000, 1, 64, 72)
    workspace = torch.empty(size + 16, dtype=torch.uint8, device=DEV)
    for at, given in ((None, size), (workspace.data_ptr(), size - 1), (workspace.data_ptr() + 4, size)):
        assert lib.bsp_grouped_weight_grad(x.data_ptr(), 64, grad.data_ptr(), 72, offsets.data_ptr(), 0, 5000, 1, 64, 72,
                                           out.data_ptr(), 1, at, given, None,
                                           _cabi.stream_handle(x.device)) == _cabi.ERR_INVALID_ARG
    torch.cuda.synchronize()
    assert bool((out == 3.0).all())


@pytest.mark.parametrize("groups", [1, 64])
def test_weight_gradient_of_very_many_rows(groups):
    """A wait for a whole contraction may last longer than the second after which one that makes no progress ends.
    One group of 2^29 rows and 13 more: its weight gradient is one tile, 8.4 million steps and 2.7 seconds long where
    63 other groups (without rows) leave too few pairs for parts, and in 74 parts where there is no other group.
    Values are 1 or -1, repeated from 2^20 rows, so that every partial sum is an integer below 2^24 and the sums are
    exact; one rounding."""
    import blksprs_b200 as bs
    from blksprs_b200.plan import check_device_status
    part, times, rest = 2 ** 20, 512, 13
    gen = torch.Generator().manual_seed(5)
    x, grad, w = ((torch.randint(0, 2, shape, generator=gen) * 2 - 1).to(BF16).to(DEV)
                  for shape in ((part, 8), (part, 8), (groups, 8, 8)))
    w.requires_grad_()
    products = x.double()[:, :, None] * grad.double()[:, None, :]
    assert products.cumsum(0).abs().max() * times < 2 ** 24
    want = products.sum(0) * times + products[:rest].sum(0)
    forward = (x.double() @ w[0].detach().double()).to(BF16)
    del products
    long = torch.cat([x.repeat(times, 1), x[:rest]]).requires_grad_()
    offsets = torch.tensor([0] + [long.shape[0]] * groups, device=DEV)
    out = bs.ops.grouped_matmul(long, w, offsets)
    for i in (0, 1, times // 2, times - 1):
        assert torch.equal(out[i * part:(i + 1) * part], forward)
    assert torch.equal(out[times * part:], forward[:rest])
    out.backward(torch.cat([grad.repeat(times, 1), grad[:rest]]))
    check_device_status()
    assert torch.equal(w.grad[0], want.to(BF16)) and not w.grad[1:].any()
    last = (grad.double() @ w[0].detach().double().T).to(BF16)
    assert torch.equal(long.grad[(times - 1) * part:times * part], last)
    assert torch.equal(long.grad[times * part:], last[:rest])


def test_layer_of_experts_with_its_gradients():
    """Two products with an activation between, forward and backward, on whole numbers small enough that fp16 holds
    every product, sum and gradient exactly: all of them have to be equal."""
    import blksprs_b200 as bs
    gen = torch.Generator().manual_seed(13)
    offsets = bounds_of([7, 0, 5, 4], 2).to(DEV)

    def small(*shape):
        return torch.randint(-1, 2, shape, generator=gen).to(FP16).to(DEV)

    x, up, down, grad = small(20, 32), small(4, 32, 40), small(4, 40, 24), small(20, 24)

    def gradients(product, dtype):
        leaves = [t.to(dtype).requires_grad_(True) for t in (x, up, down)]
        hidden = torch.relu(product(leaves[0], leaves[1]))
        out = product(hidden, leaves[2])
        return [out, *torch.autograd.grad(out, leaves, grad.to(dtype))]

    def by_mask(a, b):
        row = torch.arange(20, device=DEV)
        group = (row[:, None] >= offsets[None, :-1]) & (row[:, None] < offsets[None, 1:])
        return torch.einsum("te,tk,ekn->tn", group.to(a.dtype), a, b)

    for got, want in zip(gradients(lambda a, b: bs.ops.grouped_matmul(a, b, offsets), FP16),
                         gradients(by_mask, torch.float64)):
        assert torch.equal(got.double(), want)


def test_autocast_and_no_grad():
    import blksprs_b200 as bs
    x, w, grad, offsets = make([10, 30], 64, 72, FP32)
    with torch.autocast("cuda", dtype=BF16):
        out = bs.ops.grouped_matmul(x, w, offsets)
    assert out.dtype == BF16 and torch.equal(out, bs.ops.grouped_matmul(x.to(BF16), w.to(BF16), offsets))
    x = x.to(BF16).requires_grad_(True)
    with torch.no_grad():
        assert not bs.ops.grouped_matmul(x, w.to(BF16), offsets).requires_grad


def test_marked_tensors_and_compiled_calls():
    """Tensor subclasses (the compressed-tensor marker) and calls from a compiled function give the same values."""
    import blksprs_b200 as bs
    x, w, grad, offsets = make([10, 30], 64, 72, BF16)
    want = bs.ops.grouped_matmul(x, w, offsets)
    got = bs.ops.grouped_matmul(bs.BlksprsTensor.wrap(x), torch.nn.Parameter(w), offsets)
    assert type(got) is torch.Tensor and torch.equal(got, want)
    compiled = torch.compile(lambda a, b, c: bs.ops.grouped_matmul(a + 0, b, c) + 0, backend="eager")
    assert torch.equal(compiled(x, w, offsets), want)


def test_same_inputs_same_bits():
    import blksprs_b200 as bs
    x, w, grad, offsets = make([500, 3, 1000, 41], 520, 264, BF16)
    x.requires_grad_(True), w.requires_grad_(True)

    def step():
        out = bs.ops.grouped_matmul(x, w, offsets)
        return (out.detach(), *torch.autograd.grad(out, (x, w), grad))
    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))


# ---- 8 bits ----------------------------------------------------------------------------------------

def blocked(t, dims):
    for d in dims:
        t = t.repeat_interleave(128, d)
    return t


def plain_scaled(x, sx, w, sw, offsets):
    """64-bit product of what the 8-bit values and their scales stand for, and the same of magnitudes."""
    xd = x.double() * blocked(sx.double(), (1,))[:, :x.shape[1]]
    wd = w.double() * blocked(sw.double(), (1, 2))[:, :w.shape[1], :w.shape[2]]
    return plain(xd, wd, offsets), plain(xd.abs(), wd.abs(), offsets)


def make_scaled(sizes, depth, cols, tx=E4M3, tw=E4M3, seed=0, before=0, behind=0):
    gen = torch.Generator().manual_seed(seed)
    rows = before + sum(sizes) + behind
    x = (torch.randn((rows, depth), generator=gen)).to(tx).to(DEV)
    w = (torch.randn((len(sizes), cols, depth), generator=gen)).to(tw).to(DEV).transpose(1, 2)
    sx = torch.exp(torch.randn((rows, -(-depth // 128)), generator=gen)).to(DEV)
    sw = torch.exp(torch.randn((len(sizes), -(-depth // 128), -(-cols // 128)), generator=gen)).to(DEV)
    return x, sx, w, sw, bounds_of(sizes, before).to(DEV)


def check_scaled(x, sx, w, sw, offsets, out_dtype):
    import blksprs_b200 as bs
    got = bs.ops.grouped_matmul_scaled(x, sx, w, sw, offsets, out_dtype=out_dtype)
    assert got.dtype == out_dtype
    assert_near(got, *plain_scaled(x, sx, w, sw, offsets), x.shape[1] + 4)
    from blksprs_b200.plan import check_device_status
    check_device_status()


@pytest.mark.parametrize("out_dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("sizes", [[1], [31, 0, 33], [257, 1, 255, 0, 256], [700]], ids=str)
def test_scaled_sizes_of_groups(sizes, out_dtype):
    check_scaled(*make_scaled(sizes, 272, 136, seed=len(sizes), before=2, behind=3), out_dtype)


@pytest.mark.parametrize("seed", range(12))
def test_random_sizes(seed):
    """Sizes, strides of storage and types by chance, over both kernels of either product."""
    import random
    rng = random.Random(seed)
    groups = rng.choice((1, 2, 5, 17, 64))
    mean = rng.choice((1, 3, 20, 45, 70, 200, 600))
    sizes = [rng.choice((0, 1, rng.randint(0, 2 * mean))) for _ in range(groups)]
    before, behind = rng.choice((0, 1, 37)), rng.choice((0, 1, 260))
    depth, cols = 8 * rng.randint(1, 150), 8 * rng.randint(1, 150)
    check_training(*make(sizes, depth, cols, rng.choice((BF16, FP16)), seed, before, behind, rng.choice(("kn", "nk"))))
    check_scaled(*make_scaled(sizes, 16 * rng.randint(1, 75), cols, rng.choice((E4M3, E5M2)), rng.choice((E4M3, E5M2)),
                              seed, before, behind), rng.choice((BF16, FP16, FP32)))


@pytest.mark.parametrize("tx,tw", [(E4M3, E4M3), (E5M2, E4M3), (E4M3, E5M2), (E5M2, E5M2)],
                         ids=["e4m3", "e5m2-e4m3", "e4m3-e5m2", "e5m2"])
@pytest.mark.parametrize("depth,cols", [(16, 8), (128, 128), (144, 264), (1040, 72), (512, 392)])
def test_scaled_depths_columns_and_types(depth, cols, tx, tw):
    check_scaled(*make_scaled([37, 0, 300], depth, cols, tx, tw, seed=depth), BF16)


def test_scaled_strides():
    x, sx, w, sw, offsets = make_scaled([40, 93], 256, 136, seed=1)
    wide = torch.zeros((133, 300 + 20), dtype=E4M3, device=DEV)
    wide.view(torch.uint8)[:, 16:272] = x.view(torch.uint8)
    for xs in (wide[:, 16:272], x.view(torch.uint8).t().contiguous().t().view(E4M3)):
        assert torch.equal(xs.float(), x.float())
        check_scaled(xs, sx.t().contiguous().t(), w, sw.transpose(1, 2).contiguous().transpose(1, 2), offsets, BF16)
    check_scaled(x, sx[:, :1].expand(-1, 2), w.contiguous(), sw[:1].expand(2, -1, -1), offsets, FP32)


def test_scaled_non_finite_scale_stays_in_its_row():
    import blksprs_b200 as bs
    x, sx, w, sw, offsets = make_scaled([40, 93], 256, 136, seed=2, behind=4)
    clean = bs.ops.grouped_matmul_scaled(x, sx, w, sw, offsets)
    sx[50, 1], sx[-1] = float("nan"), float("inf")
    out = bs.ops.grouped_matmul_scaled(x, sx, w, sw, offsets)
    keep = torch.arange(x.shape[0], device=DEV) != 50
    assert out[50].isnan().all() and torch.equal(out[keep], clean[keep])


def plain_scale(largest, to):
    """The product with the reciprocal of the type's largest value, each rounded once."""
    reciprocal = torch.tensor(1.0 / LARGEST[to], dtype=torch.float32, device=largest.device)
    return (largest * reciprocal).clamp(min=2.0 ** -126)


def plain_quantize(t, largest, scale, dtype):
    """32-bit rounding of what a scale stands for, one elementary step after the other."""
    return (t.float() / scale).clamp(-largest, largest).to(dtype)


@pytest.mark.parametrize("to", [E4M3, E5M2], ids=["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 128), (7, 129), (33, 200), (5, 1040), (130, 7), (300, 512)])
def test_quantize_rows(rows, width, dtype, to):
    import blksprs_b200 as bs
    gen = torch.Generator().manual_seed(width)
    x = values(rows, width, dtype=dtype, gen=gen)
    x[0, 0] = 0.0 if width == 1 else x[0, 0]
    q, scale = bs.ops.quantize_rows(x, to)
    assert q.dtype == to and q.shape == x.shape and scale.shape == (rows, -(-width // 128))
    padded = torch.zeros((rows, 128 * scale.shape[1]), device=DEV)
    padded[:, :width] = x.float()
    want = plain_scale(padded.reshape(rows, -1, 128).abs().amax(2), to)
    assert torch.equal(scale, want)
    want_q = plain_quantize(x, LARGEST[to], blocked(want, (1,))[:, :width], to)
    assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))


@pytest.mark.parametrize("to", [E4M3, E5M2], ids=["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("depth,cols", [(1, 1), (128, 128), (130, 257), (40, 264), (272, 56)])
@pytest.mark.parametrize("order", ["kn", "nk", "strided"])
def test_quantize_blocks(depth, cols, order, dtype, to):
    import blksprs_b200 as bs
    gen = torch.Generator().manual_seed(depth)
    if order == "kn":
        w = values(3, depth, cols, dtype=dtype, gen=gen)
    elif order == "nk":
        w = values(3, cols, depth, dtype=dtype, gen=gen).transpose(1, 2)
    else:
        w = values(3, 2 * depth, 2 * cols + 1, dtype=dtype, gen=gen)[:, ::2, 1::2]
    q, scale = bs.ops.quantize_blocks(w, to)
    kb, nb = -(-depth // 128), -(-cols // 128)
    assert q.dtype == to and q.shape == w.shape and scale.shape == (3, kb, nb)
    assert q.transpose(1, 2).is_contiguous()
    padded = torch.zeros((3, kb * 128, nb * 128), device=DEV)
    padded[:, :depth, :cols] = w.float()
    want = plain_scale(padded.reshape(3, kb, 128, nb, 128).abs().amax((2, 4)), to)
    assert torch.equal(scale, want)
    want_q = plain_quantize(w, LARGEST[to], blocked(want, (1, 2))[:, :depth, :cols], to)
    assert torch.equal(q.contiguous().view(torch.uint8), want_q.contiguous().view(torch.uint8))


@pytest.mark.parametrize("to", [E4M3, E5M2], ids=["e4m3", "e5m2"])
def test_quantize_all_magnitudes(to):
    """Blocks from the smallest to the largest fp32 magnitudes, values of a block down to 2^-40 of its largest: the
    quotient is the correctly rounded one on both ways to it."""
    import blksprs_b200 as bs
    gen = torch.Generator().manual_seed(21)
    exponent = torch.arange(-149, 127).repeat_interleave(4).double()
    x = torch.randn((exponent.numel(), 128), generator=gen).clamp(-1.9, 1.9).double()
    x = x * 2.0 ** (exponent[:, None] - 40.0 * torch.rand(x.shape, generator=gen).double() ** 3)
    x = x.to(FP32).to(DEV)
    q, scale = bs.ops.quantize_rows(x, to)
    want = plain_scale(x.abs().amax(1, keepdim=True), to)
    assert torch.equal(scale, want)
    assert torch.equal(q.view(torch.uint8), plain_quantize(x, LARGEST[to], want, to).view(torch.uint8))
    q, scale = bs.ops.quantize_blocks(x.reshape(-1, 128, 1), to)
    assert torch.equal(scale.reshape(-1, 1), want)
    assert torch.equal(q.reshape(x.shape).view(torch.uint8), plain_quantize(x, LARGEST[to], want, to).view(torch.uint8))


def test_quantize_edge_values():
    import blksprs_b200 as bs
    x = torch.zeros((6, 256), device=DEV)
    x[1, 5], x[2, 5], x[3, 5], x[4, 5] = float("nan"), float("inf"), 1e-44, 3.4e38
    x[1:5, 6] = -1.0
    q, scale = bs.ops.quantize_rows(x)
    assert float(scale[0, 0]) == 2.0 ** -126 and not q[0].float().any()
    assert scale[1, 0].isnan() and q[1, :128].float().isnan().all()
    assert scale[2, 0].isinf() and q[2, 5].float().isnan() and not q[2, 6].float().any()
    assert float(scale[3, 0]) == float(plain_scale(torch.ones(1), E4M3))
    assert q[4, 5].float() == 448.0 and scale[4, 0].isfinite()
    assert (scale[:, 1] == 2.0 ** -126).all() and not q[:, 128:].float().any()
    q, scale = bs.ops.quantize_rows(x[:0])
    assert q.shape == (0, 256) and scale.shape == (0, 2)
    q, scale = bs.ops.quantize_blocks(x[None, :0])
    assert q.shape == (1, 0, 256) and scale.shape == (1, 0, 2)


def test_quantized_layer_of_experts():
    """The three together, as a served layer of experts uses them: weights rounded once, rows on every call, one
    launch for all experts.  Rounding is off by at most half a step of the value (e4m3: 2^-4 relative) plus half the
    type's smallest step (2^-10) times the scale, for each operand."""
    import blksprs_b200 as bs
    x, w, _, offsets = make([3, 130, 0, 61], 400, 264, BF16, seed=9, behind=6)
    wq, sw = bs.ops.quantize_blocks(w)
    xq, sx = bs.ops.quantize_rows(x)
    check_scaled(xq, sx, wq, sw, offsets, BF16)
    got = bs.ops.grouped_matmul_scaled(xq, sx, wq, sw, offsets).double()
    ex = x.double().abs() * 2.0 ** -4 + 2.0 ** -10 * blocked(sx.double(), (1,))[:, :400]
    ew = w.double().abs() * 2.0 ** -4 + 2.0 ** -10 * blocked(sw.double(), (1, 2))[:, :400, :264]
    allowed = plain(ex, w.abs(), offsets) + plain(x.abs(), ew, offsets) + plain(ex, ew, offsets)
    want = plain(x, w, offsets)
    magnitudes = plain(x.abs(), w.abs(), offsets) + allowed
    allowed = allowed + 404 * 2.0 ** -23 * magnitudes + half_step(BF16) * magnitudes
    assert bool(((got - want).abs() <= allowed).all())
    assert not got[-6:].any()
