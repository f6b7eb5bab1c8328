"""Measured cases of the expert-layer products: bf16 products grouped by
expert with their gradients, and microscaled 4-bit (MXFP4) quantisation and
products.

``run`` computes each case in plain 32-bit torch operations, or, where ``own``
is true, through ``kernel_mcts_b200.grouped`` and ``kernel_mcts_b200.mxfp4``.
Rows of group ``e`` are ``ends[e-1]`` (0 for the first) up to ``ends[e]``;
rows behind the last end belong to nobody and come out as zeros.
"""

import sys
from pathlib import Path

import torch

_PACKAGE = str(Path(__file__).resolve().parent.parent / "gpu-kernel-mcts_b200")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def _case(name, op, **sizes):
    """groups (0: a dense product), rows, pad (rows behind the last group), n and k (the weight is n x k), dtype."""
    case = {"name": name, "op": op, "groups": 0, "rows": 1, "pad": 0, "n": 0, "k": 0, "dtype": "bfloat16"}
    case.update(sizes)
    return case


def listed():
    return [
        # One token sent to two of eight experts: the latency of a single decode step.
        _case("grouped_token", "forward", groups=8, rows=2, n=4096, k=4096),
        # A decode batch over many experts, a few rows each: bound by reading the weights.
        _case("grouped_decode", "forward", groups=64, rows=256, n=2048, k=4096),
        # A training or prefill batch of an expert layer.
        _case("grouped_forward", "forward", groups=16, rows=8192, n=4096, k=4096),
        # Its input gradient: the same weights, contracted over their rows; a batch padded to a fixed size.
        _case("grouped_input_grad", "input_grad", groups=16, rows=8192, pad=57, n=4096, k=4096),
        # Its weights' gradient: the contracted length is each expert's row count.
        _case("grouped_wgrad", "wgrad", groups=16, rows=8192, n=4096, k=4096),
        # The weights' gradient of a micro-batch, kept in fp32 as a main gradient: bound by writing it.
        _case("grouped_wgrad_micro", "wgrad", groups=32, rows=500, n=1024, k=2048, dtype="float32"),
        # A whole training step through autograd, odd sizes throughout.
        _case("grouped_step", "step", groups=7, rows=1111, pad=9, n=1000, k=776),
        # Activations of a few tokens to four bits and back: latency.
        _case("mxfp4_round_tokens", "round", rows=3, k=4096, dtype="float16"),
        # A large weight or activation to four bits and back: memory bandwidth.
        _case("mxfp4_round", "round", rows=16384, k=8192),
        # A decode batch through a 4-bit layer, activations quantised on the way.
        _case("mxfp4_decode", "layer", rows=4, n=8192, k=8192),
        # Expert weights in four bits, a serving batch quantised on the way.
        _case("mxfp4_experts", "layer", groups=32, rows=1500, n=2048, k=4096),
        # The largest: a prefill batch, both operands in four bits.
        _case("mxfp4_prefill", "product", rows=8192, n=8192, k=8192),
    ]


def _log_int(rng, low, high, step=1):
    value = low * (high / low) ** rng.random()
    return max(low, min(high, int(round(value / step)) * step))


def draw(rng):
    op = rng.choice(["forward", "input_grad", "wgrad", "step", "round", "layer", "product"])
    if op == "round":
        return _drop_name(_case("", op, rows=_log_int(rng, 1, 16384), k=_log_int(rng, 32, 8192, 32),
                                dtype=rng.choice(sorted(DTYPES))))
    rows = _log_int(rng, 1, 8192)
    if op in ("layer", "product"):
        groups = rng.choice([0, _log_int(rng, 1, 64)])
        n, k = _log_int(rng, 64, 8192), _log_int(rng, 64, 8192, 32)
    else:
        groups = _log_int(rng, 1, 64)
        # Rows of a weight start on 16 bytes for the tensor cores; the column count of a forward product may be odd.
        n, k = _log_int(rng, 64, 4096, 1 if op == "forward" else 8), _log_int(rng, 64, 4096, 8)
    while groups * n * k > 1 << 29:
        groups = max(1, groups // 2)
    dtype = rng.choice(["bfloat16", "float32"]) if op == "wgrad" and rows <= 1024 else "bfloat16"
    pad = rng.choice([0, 0, rng.randrange(1, 200)]) if groups else 0
    return _drop_name(_case("", op, groups=groups, rows=rows, pad=pad, n=n, k=k, dtype=dtype))


def _drop_name(case):
    del case["name"]
    return case


# ------------------------------------------------------------------- inputs


def _group_ends(case, gen):
    """Row counts of a skewed router (log-normal expert popularity): some
    experts get several times the mean, some get nothing."""
    weights = torch.exp(0.5 * torch.randn(case["groups"], generator=gen, device="cuda"))
    chosen = torch.multinomial(weights, case["rows"], replacement=True, generator=gen)
    counts = torch.bincount(chosen, minlength=case["groups"])
    return torch.cumsum(counts, 0).to(torch.int32), int(counts.max())


def _fp4(rows_shape, k, gen):
    """Random 4-bit codes (two a byte, the even element in the low half) and
    E8M0 scales around one, as weights quantised earlier."""
    codes = torch.randint(0, 256, (*rows_shape, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = torch.randint(119, 125, (*rows_shape, k // 32), generator=gen, device="cuda", dtype=torch.uint8)
    return codes, scales


def _activations(rows, k, gen, dtype=torch.bfloat16):
    """N(0, 1) with channels of different magnitude, as activations have."""
    gain = torch.exp(torch.randn(k, generator=gen, device="cuda"))
    return (torch.randn(rows, k, generator=gen, device="cuda") * gain).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, groups, n, k = case["op"], case["groups"], case["n"], case["k"]
    total = case["rows"] + case["pad"]
    state = {"op": op, "groups": groups, "dtype": DTYPES[case["dtype"]], "ends": None, "most": total}
    if groups:
        state["ends"], state["most"] = _group_ends(case, gen)
    if op in ("forward", "wgrad", "step"):
        state["x"] = torch.randn(total, k, generator=gen, device="cuda").to(torch.bfloat16)
    if op in ("input_grad", "wgrad", "step"):
        state["dy"] = torch.randn(total, n, generator=gen, device="cuda").to(torch.bfloat16)
    if op in ("forward", "input_grad", "step"):
        w = torch.randn(groups, n, k, generator=gen, device="cuda", dtype=torch.bfloat16)
        state["w"] = w.mul_(k ** -0.5)
    if op == "step":
        state["x"].requires_grad_()
        state["w"].requires_grad_()
    if op in ("round", "layer"):
        state["x"] = _activations(total, k, gen, state["dtype"])
    if op == "product":
        state["a"] = _fp4((total,), k, gen)
    if op in ("layer", "product"):
        state["b"] = _fp4((groups, n) if groups else (n,), k, gen)
    state["table"] = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    return state


# --------------------------------------------------------------- plain forms


def _slots(ends, total, most):
    """Where each row stands in a [groups, most] layout, and groups * most for
    rows behind the last group."""
    rows = torch.arange(total, device=ends.device)
    bounds = torch.cat([ends.new_zeros(1), ends]).long()
    group = torch.bucketize(rows, bounds[1:], right=True)
    behind = group == ends.numel()
    return torch.where(behind, ends.numel() * most, group * most + rows - bounds[group.clamp(max=ends.numel() - 1)])


def _spread(x, slots, groups, most):
    out = x.new_zeros(groups * most + 1, x.shape[1])
    out[slots] = x
    return out[:-1].view(groups, most, -1)


def _collect(y, slots):
    flat = y.reshape(-1, y.shape[2])
    return torch.cat([flat, flat.new_zeros(1, flat.shape[1])])[slots]


def _grouped(x, w, ends, most, transpose):
    """x [rows, c] times each row's own w[e] ([n, c] transposed, or [c, n])."""
    slots = _slots(ends, x.shape[0], most)
    y = torch.bmm(_spread(x, slots, w.shape[0], most), w.transpose(1, 2) if transpose else w)
    return _collect(y, slots)


def _grouped_wgrad(dy, x, ends, most):
    slots = _slots(ends, x.shape[0], most)
    groups = ends.numel()
    behind = (slots == groups * most)[:, None]
    dy, x = dy.masked_fill(behind, 0), x.masked_fill(behind, 0)
    return torch.bmm(_spread(dy, slots, groups, most).transpose(1, 2), _spread(x, slots, groups, most))


def _fp4_values(codes, scales, table):
    values = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1).flatten(-2)
    blocks = values.unflatten(-1, (-1, 32))
    return torch.ldexp(blocks, (scales.int() - 127)[..., None]).flatten(-2)


def _fp4_round(x):
    """x in the nearest MXFP4 values, ties to the even code."""
    blocks = x.float().unflatten(-1, (-1, 32))
    largest = blocks.abs().amax(-1, keepdim=True)
    exponent = (torch.frexp(largest).exponent - 3).clamp(-127, 127)
    exponent = torch.where(largest == 0, -127, exponent)
    scaled = torch.ldexp(blocks, -exponent)
    size = scaled.abs().clamp(max=6)
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    rounded = torch.copysign(torch.round(size / step) * step, scaled)
    return torch.ldexp(rounded, exponent).flatten(-2)


def run(state):
    op, ends, most = state["op"], state["ends"], state["most"]
    if own:
        return _run_own(state)
    if op == "forward":
        return _grouped(state["x"].float(), state["w"].float(), ends, most, True).to(torch.bfloat16)
    if op == "input_grad":
        return _grouped(state["dy"].float(), state["w"].float(), ends, most, False).to(torch.bfloat16)
    if op == "wgrad":
        return _grouped_wgrad(state["dy"].float(), state["x"].float(), ends, most).to(state["dtype"])
    if op == "step":
        x, w, dy = state["x"].detach().float(), state["w"].detach().float(), state["dy"].float()
        outs = (_grouped(x, w, ends, most, True), _grouped(dy, w, ends, most, False), _grouped_wgrad(dy, x, ends, most))
        return tuple(t.to(torch.bfloat16) for t in outs)
    if op == "round":
        return _fp4_round(state["x"]).to(torch.bfloat16)
    a = _fp4_round(state["x"]) if op == "layer" else _fp4_values(*state["a"], state["table"])
    b = _fp4_values(*state["b"], state["table"])
    y = a @ b.T if ends is None else _grouped(a, b, ends, most, True)
    return y.to(torch.bfloat16)


def _run_own(state):
    from kernel_mcts_b200 import grouped, mxfp4

    op, ends = state["op"], state["ends"]
    if op == "forward":
        return grouped.grouped_gemm(state["x"], state["w"], ends)
    if op == "input_grad":
        return grouped.grouped_gemm(state["dy"], state["w"], ends, w_layout="row")
    if op == "wgrad":
        return grouped.grouped_gemm_wgrad(state["dy"], state["x"], ends, dtype=state["dtype"])
    if op == "step":
        y = grouped.grouped_linear(state["x"], state["w"], ends)
        return (y.detach(), *torch.autograd.grad(y, (state["x"], state["w"]), state["dy"]))
    if op == "round":
        return mxfp4.mxfp4_dequantize(mxfp4.mxfp4_quantize(state["x"]), dtype=torch.bfloat16)
    a = mxfp4.mxfp4_quantize(state["x"]) if op == "layer" else mxfp4.MXFP4Tensor(*state["a"])
    return mxfp4.mxfp4_gemm(a, mxfp4.MXFP4Tensor(*state["b"]), ends)


# ------------------------------------------------------------- cost and truth


def work(case):
    """Each input read once, each output written once; of the experts, those
    that a uniform router would be expected to use."""
    op, groups, rows, n, k = case["op"], case["groups"], case["rows"], case["n"], case["k"]
    total = rows + case["pad"]
    used = groups * (1 - (1 - 1 / groups) ** rows) if groups else 1
    product = 2 * rows * n * k
    fp4 = k / 2 + k / 32  # bytes of one quantised row
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    if op == "round":
        return {"bytes": int(rows * (k * size + 2 * fp4 + 2 * k)), "flops": 8 * rows * k}
    if op == "forward":
        return {"bytes": int(2 * (rows * k + used * n * k + total * n)), "flops": product}
    if op == "input_grad":
        return {"bytes": int(2 * (rows * n + used * n * k + total * k)), "flops": product}
    if op == "wgrad":
        return {"bytes": int(2 * rows * (n + k) + size * groups * n * k), "flops": product}
    if op == "step":
        return {"bytes": int(2 * (rows * (n + k) + total * (n + k) + (used + groups) * n * k)), "flops": 3 * product}
    inputs = total * 2 * k if op == "layer" else rows * fp4
    return {"bytes": int(inputs + used * n * fp4 + 2 * total * n), "flops": product}


def _exact_values(codes, scales):
    """Values of MXFP4 codes from their bits: sign, two exponent bits, one mantissa bit."""
    pair = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int64)
    exponent, mantissa = (pair >> 1) & 3, (pair & 1).double()
    size = torch.where(exponent == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * 2.0 ** (exponent - 1).double())
    values = torch.where(pair >= 8, -size, size)
    return values * (2.0 ** (scales.double() - 127)).repeat_interleave(32, -1)


def _exact_round(x):
    """The nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 by counting the midpoints
    below, those between an odd code and the next even one included."""
    blocks = x.double().unflatten(-1, (-1, 32))
    largest = blocks.abs().amax(-1, keepdim=True)
    # The exponent field of a double is floor(log2) exactly, which log2 itself is not at every power of two.
    scale = 2.0 ** ((largest.view(torch.int64) >> 52) - 1025).clamp(-127, 127).double()
    size = blocks.abs() / scale
    code = ((size > 0.25).int() + (size >= 0.75) + (size > 1.25) + (size >= 1.75) + (size > 2.5) + (size >= 3.5) + (size > 5))
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    return (levels[code.long()] * scale * torch.sign(blocks)).flatten(-2)


def exact(case, seed):
    state = prepare(case, seed)
    op, ends = state["op"], state["ends"]
    bounds = [0, *ends.tolist()] if ends is not None else [0, state["most"]]

    def by_group(a, b, times):
        out = None
        for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
            part = times(a[lo:hi].double(), b[e].double())
            out = part.new_zeros(a.shape[0], part.shape[1]) if out is None else out
            out[lo:hi] = part
        return out

    def forward(x, w):
        return by_group(x, w, lambda r, m: r @ m.T)

    def input_grad(dy, w):
        return by_group(dy, w, lambda r, m: r @ m)

    def wgrad(dy, x):
        return torch.stack([dy[lo:hi].double().T @ x[lo:hi].double() for lo, hi in zip(bounds, bounds[1:])])

    if op == "forward":
        return forward(state["x"], state["w"])
    if op == "input_grad":
        return input_grad(state["dy"], state["w"])
    if op == "wgrad":
        return wgrad(state["dy"], state["x"])
    if op == "step":
        x, w = state["x"].detach(), state["w"].detach()
        return forward(x, w), input_grad(state["dy"], w), wgrad(state["dy"], x)
    if op == "round":
        return _exact_round(state["x"])
    a = _exact_round(state["x"]) if op == "layer" else _exact_values(*state["a"])
    b = state["b"] if ends is not None else tuple(t[None] for t in state["b"])
    values = torch.stack([_exact_values(c, s).float() for c, s in zip(*b)])  # exact: at most 2 bits times 2^e
    return forward(a, values)
