"""Calls of the grouped products and the 8-bit rounding that are refused, on the CPU: every refusal comes before
anything is launched, and the last of them is that the tensors are not on a GPU."""
import pytest
import torch

import blksprs_b200 as bs
from blksprs_b200 import _cabi

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn


def operands(rows=6, depth=16, cols=24, groups=3, dtype=BF16):
    return (torch.zeros((rows, depth), dtype=dtype), torch.zeros((groups, depth, cols), dtype=dtype),
            torch.zeros(groups + 1, dtype=torch.int32))


def scaled_operands(rows=6, depth=144, cols=136, groups=2, dtype=F8):
    x, w, offsets = operands(rows, depth, cols, groups, torch.float32)
    return [x.to(dtype), torch.ones((rows, 2)), w.to(dtype), torch.ones((groups, 2, 2)), offsets]


@pytest.mark.parametrize("change,message", [
    (lambda x, w, o: (x[None], w, o), "2 dimensions"),
    (lambda x, w, o: (x, w[0], o), "3 dimensions"),
    (lambda x, w, o: (x.float(), w, o), "float16 or bfloat16"),
    (lambda x, w, o: (x.to(F8), w, o), "float16 or bfloat16"),
    (lambda x, w, o: (x, w.half(), o), "same dtype"),
    (lambda x, w, o: (x, w, o.float()), "int32 or int64"),
    (lambda x, w, o: (x, w, o[:-1]), "one entry more"),
    (lambda x, w, o: (x, w, o[None]), "one entry more"),
    (lambda x, w, o: (x, w, torch.zeros(8, dtype=torch.int32)[::2]), "contiguous"),
    (lambda x, w, o: (x[:, :8], w, o), "Inner dimensions"),
    (lambda x, w, o: (x[:, :12], w[:, :12], o), "divisible"),
    (lambda x, w, o: (x, w[:, :, :20], o), "divisible"),
    (lambda x, w, o: (x, w[:1].expand(1025, -1, -1), torch.zeros(1026, dtype=torch.int32)), "at most 1024"),
    (lambda x, w, o: (x, w, o), "must be on GPU"),
])
def test_grouped_matmul_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        bs.ops.grouped_matmul(*change(*operands()))


@pytest.mark.parametrize("change,message", [
    (lambda a: a.__setitem__(0, a[0].to(BF16)), "float8_e4m3fn or float8_e5m2"),
    (lambda a: a.__setitem__(2, a[2].to(BF16)), "float8_e4m3fn or float8_e5m2"),
    (lambda a: a.__setitem__(1, a[1].double()), "float32"),
    (lambda a: a.__setitem__(3, a[3].half()), "float32"),
    (lambda a: a.__setitem__(1, a[1][:, :1]), "Scale shape"),
    (lambda a: a.__setitem__(1, a[1][:5]), "Scale shape"),
    (lambda a: a.__setitem__(3, a[3][:, :, :1]), "Scale shape"),
    (lambda a: a.__setitem__(3, a[3][:1]), "Scale shape"),
    (lambda a: a.__setitem__(1, a[1].requires_grad_(True)), "no gradient"),
    (lambda a: (a.__setitem__(0, a[0][:, :136]), a.__setitem__(2, a[2][:, :136])), "divisible by 16"),
    (lambda a: None, "must be on GPU"),
])
def test_grouped_matmul_scaled_refuses(change, message):
    arguments = scaled_operands()
    change(arguments)
    with pytest.raises(ValueError, match=message):
        bs.ops.grouped_matmul_scaled(*arguments)


def test_switched_off_validation_still_refuses_what_would_be_read_out_of_bounds():
    x, w, offsets = operands()
    bs.utils.disable_validation()
    try:
        for bad in ((x[:, :8], w, offsets), (x, w, offsets[:-1]), (x, w.half(), offsets), (x, w[0], offsets),
                    (x, w, offsets), (x[0], w, offsets), (x, w, offsets.float())):
            with pytest.raises(ValueError):
                bs.ops.grouped_matmul(*bad)
        arguments = scaled_operands()
        for at, bad in ((1, arguments[1][:, :1]), (3, arguments[3][:1]), (0, arguments[0][:, :16]), (4, offsets)):
            with pytest.raises(ValueError):
                bs.ops.grouped_matmul_scaled(*arguments[:at], bad, *arguments[at + 1:])
        for op, t in ((bs.ops.quantize_rows, torch.zeros((4, 40))), (bs.ops.quantize_blocks, torch.zeros((2, 4, 40)))):
            for bad in (t, t[0], t.double()):
                with pytest.raises(ValueError):
                    op(bad)
    finally:
        bs.utils.enable_validation()


def test_group_limit_is_the_library_s():
    from blksprs_b200.ops import grouped_matmul  # noqa: F401  (the module's name is the function's too)
    import sys
    assert sys.modules["blksprs_b200.ops.grouped_matmul"].MAX_GROUPS == _cabi.lib().bsp_grouped_max_groups()


def test_grouped_matmul_scaled_refuses_output_types():
    with pytest.raises(ValueError, match="Output dtype"):
        bs.ops.grouped_matmul_scaled(*scaled_operands(), out_dtype=torch.float64)


@pytest.mark.parametrize("op,shape", [(bs.ops.quantize_rows, (4, 40)), (bs.ops.quantize_blocks, (2, 4, 40))])
def test_quantize_refuses(op, shape):
    t = torch.zeros(shape)
    for value, dtype, message in ((t[0], F8, "dimensions"), (t.double(), F8, "float16, bfloat16, or float32"),
                                  (t, torch.int8, "Output dtype"), (t.clone().requires_grad_(True), F8, "no gradient"),
                                  (t, F8, "must be on GPU")):
        with pytest.raises(ValueError, match=message):
            op(value, dtype)


def test_c_entries_refuse_without_a_device():
    lib, bad, unsupported, ok = _cabi.lib(), _cabi.ERR_INVALID_ARG, _cabi.ERR_UNSUPPORTED, _cabi.OK
    p = 1 << 20      # an aligned address that is never touched

    def rows(x=p, ld_x=64, w=p, sg=64 * 64, ld_w=64, inner=1, offsets=p, T=4, E=2, K=64, N=64, out=p, dtype=1):
        return lib.bsp_grouped_matmul(x, ld_x, w, sg, ld_w, inner, offsets, 0, T, E, K, N, out, dtype, None, None)

    assert rows(T=0) == ok
    for change in (dict(x=None), dict(w=p + 8), dict(out=p + 2), dict(offsets=None), dict(T=-1), dict(E=0), dict(K=0),
                   dict(K=60), dict(N=60), dict(ld_x=56), dict(ld_x=68), dict(ld_w=56), dict(sg=0), dict(sg=-8)):
        assert rows(**change) == bad, change
    for change in (dict(dtype=2), dict(dtype=3), dict(E=lib.bsp_grouped_max_groups() + 1), dict(T=1 << 31)):
        assert rows(**change) == unsupported, change

    def grad(x=p, ld_x=64, g=p, ld_g=64, offsets=p, T=4, E=2, K=64, N=64, out=p, dtype=1):
        return lib.bsp_grouped_weight_grad(x, ld_x, g, ld_g, offsets, 0, T, E, K, N, out, dtype, None, 0, None, None)

    for change in (dict(T=0), dict(x=None), dict(g=p + 4), dict(K=4), dict(N=4), dict(ld_g=32), dict(offsets=None)):
        assert grad(**change) == bad, change
    assert grad(dtype=2) == unsupported
    for sizes in ((0, 1, 64, 64), (64, 0, 64, 64), (64, 1, 0, 64), (64, 1, 64, 0), (64, 5000, 64, 64)):
        assert lib.bsp_grouped_weight_grad_workspace(*sizes) == 0

    def scaled(x=p, ld_x=64, tx=3, sx=p, w=p, sg=64 * 64, ld_w=64, tw=4, sw=p, T=4, E=2, K=64, N=64, out=p, dtype=1):
        return lib.bsp_grouped_matmul_scaled(x, ld_x, tx, sx, 1, 1, w, sg, ld_w, tw, sw, 1, 1, 1, p, 0, T, E, K, N,
                                             out, dtype, None, None)

    assert scaled(T=0) == ok
    for change in (dict(sx=None), dict(sw=None), dict(K=56), dict(ld_x=72), dict(ld_w=48), dict(N=4), dict(w=p + 8)):
        assert scaled(**change) == bad, change
    for change in (dict(tx=1), dict(tw=0), dict(dtype=3), dict(E=5000)):
        assert scaled(**change) == unsupported, change

    assert lib.bsp_quantize_rows(None, 0, 0, 128, 1, None, 3, None, None) == ok
    assert lib.bsp_quantize_rows(None, 0, 1, 128, 1, p, 3, p, None) == bad
    assert lib.bsp_quantize_rows(p, 128, 1, 128, 1, p, 1, p, None) == unsupported
    assert lib.bsp_quantize_rows(p, 128, 1, 128, 3, p, 3, p, None) == unsupported
    assert lib.bsp_quantize_blocks(p, 1, 1, 1, 1, 1, 1, 1, p + 1, 3, p, None) == bad
    assert lib.bsp_quantize_blocks(None, 1, 1, 1, 0, 1, 1, 1, None, 3, None, None) == ok
