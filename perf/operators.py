"""Workloads of the expert products: ``grouped_matmul`` (16 bits, with gradients), ``grouped_matmul_scaled``
(8 bits with a scale for each block of 128) and ``quantize_rows`` / ``quantize_blocks``, which make its operands.

A case is one call (a training step: one forward and backward) as a layer of experts makes it: the rows of a batch
are sorted by expert, ``group_offsets`` says where each expert's rows begin and end, and rows outside every group
(the padding of a batch of fixed size) belong to no expert.
"""
import math

import torch

own = False

BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32,
          "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
SMALLEST_SCALE = 2.0 ** -126

DEVICE = "cuda"


def grouped(name, rows, experts, k, n, *, train=False, dtype="bf16", stored="kn", spare=0, skew=0.5):
    return dict(name=name, op="grouped", rows=rows, experts=experts, k=k, n=n, train=train, dtype=dtype,
                stored=stored, spare=spare, skew=skew)


def scaled(name, rows, experts, k, n, *, x="e4m3", w="e4m3", out="bf16", spare=0, skew=0.5):
    return dict(name=name, op="scaled", rows=rows, experts=experts, k=k, n=n, x=x, w=w, out=out, spare=spare,
                skew=skew)


def quantized(name, rows, k, *, experts=0, dtype="bf16", to="e4m3"):
    """``experts`` = 0: the rows of a batch, a scale for each 1 x 128; else the weights of that many experts."""
    return dict(name=name, op="quantize", rows=rows, k=k, experts=experts, dtype=dtype, to=to)


def listed():
    return [
        # one token of a conversation, sent to two of eight experts
        grouped("experts, one token", 2, 8, 2048, 4096),
        # one decoding step of 64 conversations, two experts each; some experts get nothing
        grouped("experts, decoding batch", 128, 32, 4096, 2048),
        # prompts of 8192 tokens in all, two experts each, the batch padded to a fixed size
        grouped("experts, prompts", 16384, 16, 2048, 4096, spare=384),
        # many experts with short groups of every length, weights stored as torch.nn.Linear holds them
        grouped("experts, short groups", 4099, 64, 2048, 1024, stored="nk", dtype="fp16", skew=0.8),
        # a training step: forward, gradients of the rows and of every expert's weights
        grouped("experts, training", 16384, 8, 4096, 4096, train=True),
        # a training step on odd sizes, experts without a row among them
        grouped("experts, training, ragged", 1999, 33, 1032, 1496, train=True, dtype="fp16", stored="nk", spare=33,
                skew=1.0),
        # one token through one layer of 8-bit weights
        scaled("8 bits, one token", 1, 1, 4096, 4096),
        # one decoding step of 64 conversations over 8-bit experts
        scaled("8 bits, decoding batch", 128, 32, 4096, 2048),
        # prompts over 8-bit experts
        scaled("8 bits, prompts", 16384, 16, 4096, 4096),
        # odd sizes: the last scale of a row stands for 16 values, the last of a weight for 8 columns
        scaled("8 bits, ragged", 2001, 5, 1040, 1288, out="fp16", spare=47, skew=1.0),
        # the rows of a batch of prompts on their way into the 8-bit product
        quantized("quantize rows", 16384, 4096),
        # the weights of a layer of experts, once after loading or after a step of the optimizer
        quantized("quantize weights", 4096, 2048, experts=32),
    ]


def draw(rng):
    def size(low, high, step):
        return step * round(2.0 ** rng.uniform(math.log2(low / step), math.log2(high / step)))

    most = {}
    for case in listed():
        most[case["op"]] = max(most.get(case["op"], 0), _cost(case))
    while True:
        op = rng.choice(("grouped", "grouped", "scaled", "scaled", "quantize"))
        if op == "quantize":
            experts = rng.choice((0, 0, rng.randint(1, 16)))
            case = quantized(None, size(1, 32768, 1) if not experts else size(256, 4096, 8), size(256, 8192, 16),
                             experts=experts, dtype=rng.choice(("bf16", "fp16", "fp32")),
                             to=rng.choice(("e4m3", "e4m3", "e5m2")))
        else:
            rows, experts = size(1, 32768, 1), size(1, 64, 1)
            k, n = size(256, 4096, 8 if op == "grouped" else 16), size(256, 4096, 8)
            spare = rng.choice((0, 0, rng.randint(1, 500)))
            skew = round(rng.uniform(0.0, 1.0), 2)
            if op == "grouped":
                case = grouped(None, rows, experts, k, n, train=rng.random() < 0.5, dtype=rng.choice(("bf16", "fp16")),
                               stored=rng.choice(("kn", "nk")), spare=spare, skew=skew)
            else:
                case = scaled(None, rows, experts, k, n, x=rng.choice(("e4m3", "e4m3", "e5m2")),
                              w=rng.choice(("e4m3", "e4m3", "e5m2")), out=rng.choice(("bf16", "fp16", "fp32")),
                              spare=spare, skew=skew)
        if _cost(case) <= most[op]:
            del case["name"]
            return case


def _cost(case):
    """Time of a pass at a card's usual rates, to keep drawn cases below the largest listed one."""
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.5e15)


def _sizes(case, seed):
    """Rows of each expert: a random share of the rows, some experts more in demand than others."""
    g = torch.Generator().manual_seed(seed * 7919 + 17)
    demand = torch.exp(case["skew"] * torch.randn(case["experts"], generator=g, dtype=torch.float64))
    to = torch.multinomial(demand / demand.sum(), case["rows"], replacement=True, generator=g)
    return torch.bincount(to, minlength=case["experts"])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).mul_(scale).to(dtype)

    if case["op"] == "quantize":
        dtype = DTYPES[case["dtype"]]
        if case["experts"]:
            w = torch.empty((case["experts"], case["rows"], case["k"]), dtype=dtype, device=DEVICE)
            for e in range(case["experts"]):
                w[e] = normal(case["rows"], case["k"], scale=case["rows"] ** -0.5)
            return {"case": case, "w": w}
        # activations: a few channels are far larger than the others
        channels = torch.exp(normal(case["k"]))
        return {"case": case, "x": normal(case["rows"], case["k"]).mul_(channels).to(dtype)}

    sizes = _sizes(case, seed)
    offsets = torch.zeros(case["experts"] + 1, dtype=torch.int64)
    offsets[1:] = torch.cumsum(sizes, 0)
    total = case["rows"] + case["spare"]
    hit = torch.nonzero(sizes).reshape(-1)
    state = {"case": case, "offsets": offsets.to(torch.int32).to(DEVICE),
             # what the plain form needs to know of the groups on the host
             "most": int(sizes.max()), "hit": hit.to(DEVICE),
             "slot": (torch.cumsum((sizes > 0).to(torch.int64), 0) - 1).to(DEVICE)}
    experts, k, n = case["experts"], case["k"], case["n"]
    if case["op"] == "grouped":
        dtype = DTYPES[case["dtype"]]
        state["x"] = normal(total, k, dtype=dtype)
        shape = (experts, k, n) if case["stored"] == "kn" else (experts, n, k)
        w = torch.empty(shape, dtype=dtype, device=DEVICE)
        for e in range(experts):
            w[e] = normal(*shape[1:], scale=k ** -0.5)
        state["w"] = w if case["stored"] == "kn" else w.transpose(1, 2)
        if case["train"]:
            state["x"].requires_grad_(True)
            state["w"].requires_grad_(True)
            state["grad"] = normal(total, n, dtype=dtype)
        return state
    channels = torch.exp(0.5 * normal(k))
    state["x"], state["x_scale"] = _plain_rows(normal(total, k).mul_(channels), case["x"])
    w = torch.empty((experts, n, k), dtype=DTYPES[case["w"]], device=DEVICE).transpose(1, 2)
    state["w_scale"] = torch.empty((experts, -(-k // BLOCK), -(-n // BLOCK)), dtype=torch.float32, device=DEVICE)
    for e in range(experts):
        q, s = _plain_blocks(normal(1, k, n, scale=k ** -0.5), case["w"])
        w[e] = q[0]
        state["w_scale"][e] = s[0]
    state["w"] = w
    return state


# ---- the plain forms -----------------------------------------------------------------------------

def _padded(k):
    return -(-k // BLOCK) * BLOCK


def _round_to(values, scale, to):
    return (values / scale).clamp(-LARGEST[to], LARGEST[to]).to(DTYPES[to])


def _plain_rows(x, to):
    """x (rows, K) -> 8-bit values and the scale of each 1 x 128 block: its largest magnitude / the type's largest."""
    rows, k = x.shape
    padded = torch.zeros((rows, _padded(k)), dtype=torch.float32, device=x.device)
    padded[:, :k] = x.float()
    blocks = padded.reshape(rows, -1, BLOCK)
    scale = (blocks.abs().amax(2) / LARGEST[to]).clamp(min=SMALLEST_SCALE)
    q = _round_to(blocks, scale[:, :, None], to).reshape(rows, -1)[:, :k]
    return q.contiguous(), scale


def _plain_blocks(w, to):
    """w (E, K, N) -> 8-bit values and the scale of each 128 x 128 block."""
    experts, k, n = w.shape
    padded = torch.zeros((experts, _padded(k), _padded(n)), dtype=torch.float32, device=w.device)
    padded[:, :k, :n] = w.float()
    blocks = padded.reshape(experts, padded.shape[1] // BLOCK, BLOCK, padded.shape[2] // BLOCK, BLOCK)
    scale = (blocks.abs().amax((2, 4)) / LARGEST[to]).clamp(min=SMALLEST_SCALE)
    q = _round_to(blocks, scale[:, :, None, :, None], to).reshape(padded.shape)[:, :k, :n]
    return q, scale


def _places(state, total):
    """Of each row: whether it is in a group, and its place among the groups' rows padded to the longest group."""
    offsets, most = state["offsets"].long(), state["most"]
    row = torch.arange(total, device=offsets.device)
    inside = (row >= offsets[0]) & (row < offsets[-1])
    group = (row[:, None] >= offsets[None, 1:]).sum(1).clamp(max=offsets.numel() - 2)
    place = state["slot"][group] * most + row - offsets[group]
    # rows of no group share one place behind the last
    return inside, torch.where(inside, place, state["hit"].numel() * most)


def _spread(rows, place, groups, most):
    """Rows in 32 bits at their places: (groups, most, columns), zeros where a group is shorter than the longest."""
    padded = torch.zeros((groups * most + 1, rows.shape[1]), dtype=torch.float32, device=rows.device)
    padded.index_copy_(0, place, rows.float())
    return padded[:-1].reshape(groups, most, rows.shape[1])


def _collect(padded, inside, place):
    """The rows back from their places; zeros for rows of no group."""
    flat = padded.reshape(-1, padded.shape[-1])
    return torch.where(inside[:, None], flat[place.clamp(max=flat.shape[0] - 1)], 0.0)


def _plain_grouped(x, w, inside, place, state):
    """x and w in 32 bits or fewer; the product in 32."""
    return _collect(torch.bmm(_spread(x, place, state["hit"].numel(), state["most"]), w.float()), inside, place)


def _unscaled(x, scale):
    """8-bit rows times their scales."""
    return x.float() * scale.repeat_interleave(BLOCK, 1)[:, :x.shape[1]]


def _unscaled_blocks(w, scale):
    return w.float() * scale.repeat_interleave(BLOCK, 1).repeat_interleave(BLOCK, 2)[:, :w.shape[1], :w.shape[2]]


def _run_plain(state):
    case = state["case"]
    if case["op"] == "quantize":
        q, scale = _plain_blocks(state["w"], case["to"]) if case["experts"] else _plain_rows(state["x"], case["to"])
        return {"values": q.to(torch.bfloat16), "scale": scale}
    x, w, hit = state["x"].detach(), state["w"].detach(), state["hit"]
    inside, place = _places(state, x.shape[0])
    if case["op"] == "scaled":
        w_hit = _unscaled_blocks(w.view(torch.uint8)[hit].view(w.dtype), state["w_scale"][hit])
        out = _plain_grouped(_unscaled(x, state["x_scale"]), w_hit, inside, place, state)
        return {"out": out.to(DTYPES[case["out"]])}
    w_hit = w[hit].float()
    out = {"out": _plain_grouped(x, w_hit, inside, place, state).to(x.dtype)}
    if case["train"]:
        grad = state["grad"]
        out["grad_x"] = _plain_grouped(grad, w_hit.transpose(1, 2), inside, place, state).to(x.dtype)
        groups, most = hit.numel(), state["most"]
        products = torch.bmm(_spread(x, place, groups, most).transpose(1, 2), _spread(grad, place, groups, most))
        out["grad_w"] = torch.zeros_like(w).index_copy_(0, hit, products.to(w.dtype))
    return out


def _run_own(state):
    import blksprs_b200 as bs
    case = state["case"]
    if case["op"] == "quantize":
        if case["experts"]:
            q, scale = bs.ops.quantize_blocks(state["w"], DTYPES[case["to"]])
        else:
            q, scale = bs.ops.quantize_rows(state["x"], DTYPES[case["to"]])
        return {"values": q.to(torch.bfloat16), "scale": scale}
    if case["op"] == "scaled":
        return {"out": bs.ops.grouped_matmul_scaled(state["x"], state["x_scale"], state["w"], state["w_scale"],
                                                    state["offsets"], out_dtype=DTYPES[case["out"]])}
    out = bs.ops.grouped_matmul(state["x"], state["w"], state["offsets"])
    if not case["train"]:
        return {"out": out}
    grad_x, grad_w = torch.autograd.grad(out, (state["x"], state["w"]), state["grad"])
    return {"out": out.detach(), "grad_x": grad_x, "grad_w": grad_w}


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    """The rows inside groups are computed; weights of experts that get no row need not be read (counted for a
    spread of the rows over the experts that is even in the mean)."""
    size = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1, "e5m2": 1}
    k, rows, experts = case["k"], case["rows"], case["experts"]
    if case["op"] == "quantize":
        values = rows * k * max(experts, 1)
        scales = (experts * -(-rows // BLOCK) if experts else rows) * -(-k // BLOCK)
        # the values come back as 16 bits each
        return {"bytes": values * (size[case["dtype"]] + 2) + 4 * scales, "flops": 2 * values}
    n, total = case["n"], rows + case["spare"]
    hit = experts * (1.0 - (1.0 - 1.0 / experts) ** rows)
    flops = 2 * rows * k * n
    if case["op"] == "scaled":
        blocks = -(-k // BLOCK)
        return {"bytes": round(rows * (k + 4 * blocks) + hit * (k * n + 4 * blocks * -(-n // BLOCK))
                               + total * n * size[case["out"]]), "flops": flops}
    forward = rows * k + hit * k * n + total * n
    if not case["train"]:
        return {"bytes": round(2 * forward), "flops": flops}
    # rows, weights and the output's gradient read once; output and both gradients written once
    return {"bytes": round(2 * (forward + rows * n + total * k + experts * k * n)), "flops": 3 * flops}


# ---- the same from the definitions in 64 bits ------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize":
        # the 8-bit values are a rounding, not a number that more bits come nearer to
        to = LARGEST[case["to"]]
        if case["experts"]:
            scales = []
            for w in state["w"]:
                tiles = [part.double().abs().split(BLOCK, 1) for part in w.split(BLOCK, 0)]
                scales.append(torch.stack([torch.stack([t.max() for t in line]) for line in tiles]) / to)
            return {"values": None, "scale": torch.stack(scales)}
        columns = [part.double().abs().amax(1) / to for part in state["x"].split(BLOCK, 1)]
        return {"values": None, "scale": torch.stack(columns, 1)}
    bounds = state["offsets"].tolist()
    x, w = state["x"].detach(), state["w"].detach()
    total, n = x.shape[0], case["n"]
    out = torch.zeros((total, n), dtype=torch.float64, device=x.device)
    train = case["op"] == "grouped" and case["train"]
    if train:
        grad_x = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
        grad_w = torch.zeros(w.shape, dtype=torch.float64, device=x.device)
    for e, (first, last) in enumerate(zip(bounds, bounds[1:])):
        if first == last:
            continue
        rows, weight = x[first:last].double(), w[e].double()
        if case["op"] == "scaled":
            column = torch.arange(case["k"], device=x.device) // BLOCK
            rows = rows * state["x_scale"][first:last].double()[:, column]
            weight = weight * state["w_scale"][e].double()[column][:, torch.arange(n, device=x.device) // BLOCK]
        out[first:last] = rows @ weight
        if train:
            grad = state["grad"][first:last].double()
            grad_x[first:last] = grad @ weight.t()
            grad_w[e] = rows.t() @ grad
    return {"out": out, "grad_x": grad_x, "grad_w": grad_w} if train else {"out": out}
