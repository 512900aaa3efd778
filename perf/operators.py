"""Operators of a joint block on an 8-bit floating-point base, as cases that can be timed and compared.

Five operators, reached as a training or sampling program reaches them:

- ``fp8_quantize_*`` / ``fp8_decode``: a matrix to 8-bit floating point (e4m3) with a power-of-two scale
  for each 128 values of a row, of a column, or for each 128 x 128 block of a weight, and back;
- ``fp8_linear_forward``: rows quantized on the fly, times a block-scaled weight;
- ``fp8_linear_backward``: the input gradient of that product;
- ``fp8_weight_gradient``: its weight gradient, reduced over the tokens in groups of 128;
- ``rotary_table`` / ``rotary_forward`` / ``rotary_backward``: rotary positions of the query and key heads,
  with the heads' RMS norm where the block has one.

Sizes are those of the model's configurations: hidden 3072, 24 heads of 128, feed-forward 12288 or 8192
(gate and up fused: twice that), 4608 tokens for a 1024^2 picture with 512 text tokens, 17792 for a packed
batch of four, one row for the time conditions. Token counts in use are seldom round.

``run`` computes the plain form (elementary torch operations in 32 bits) while ``own`` is false, and calls
the framework where it is true.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

GROUP = 128
DIM, HEADS, HEAD_DIM, FFN = 3072, 24, 128, 12288
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
MOST_ROWS, MOST_FEATURES = 17792, 24576


def _framework():
    root = os.path.join(os.getcwd(), "moss-image_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from moss_offload import fp8_kernels, rotary

    return fp8_kernels, rotary


# ---- cases -------------------------------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # a text of 77 tokens after its projection: the call is mostly latency
        {"name": "quantize_rows_77", "kind": "quantize", "form": "rows", "rows": 77, "cols": DIM, "dtype": "float32"},
        # the feed-forward activations of a packed batch, kept in 8 bits for both of the products that read them
        {"name": "quantize_both_17792", "kind": "quantize", "form": "both", "rows": MOST_ROWS, "cols": FFN,
         "dtype": "bfloat16"},
        # the time conditions' modulation: one row a sampling step, the whole weight is read for it
        {"name": "forward_1", "kind": "forward", "rows": 1, "in": DIM, "out": 6 * DIM, "dtype": "bfloat16",
         "scales": "power", "bias": True},
        # a 256^2 picture and its text through one of the attention's projections
        {"name": "forward_333", "kind": "forward", "rows": 333, "in": DIM, "out": DIM, "dtype": "bfloat16",
         "scales": "power", "bias": False},
        # gate and up of a 1024^2 picture
        {"name": "forward_4608", "kind": "forward", "rows": 4608, "in": DIM, "out": 2 * FFN, "dtype": "bfloat16",
         "scales": "power", "bias": False},
        # the down projection of a packed batch, from a checkpoint whose block scales are any float32
        {"name": "forward_17792", "kind": "forward", "rows": MOST_ROWS, "in": FFN, "out": DIM, "dtype": "bfloat16",
         "scales": "float32", "bias": False},
        # input gradients: a small picture's projection, a 1024^2 picture's gate and up
        {"name": "backward_333", "kind": "backward", "rows": 333, "in": DIM, "out": DIM, "dtype": "bfloat16",
         "scales": "power"},
        {"name": "backward_4608", "kind": "backward", "rows": 4608, "in": DIM, "out": 2 * FFN, "dtype": "bfloat16",
         "scales": "power"},
        # weight gradients: a projection at 512^2, the down projection of the packed batch
        {"name": "weight_1333", "kind": "weight", "rows": 1333, "in": DIM, "out": DIM, "dtype": "bfloat16",
         "gradient": "float32"},
        {"name": "weight_17792", "kind": "weight", "rows": MOST_ROWS, "in": FFN, "out": DIM, "dtype": "bfloat16",
         "gradient": "bfloat16"},
        # one new token of each of 16 sequences at positions far past the trained length, neighbouring pairs,
        # half of each head, fewer key heads: table and rotation
        {"name": "rotary_step", "kind": "rotary", "batch": 16, "tokens": 1, "heads": 32, "kv_heads": 8,
         "head_dim": HEAD_DIM, "rotary_dim": 64, "layout": "interleaved", "norm": False, "backward": False,
         "factor": 8.0, "dtype": "bfloat16"},
        # the joint block's attention at 1024^2, forward and backward, with the norms of queries and keys
        {"name": "rotary_train", "kind": "rotary", "batch": 1, "tokens": 4608, "heads": HEADS, "kv_heads": HEADS,
         "head_dim": HEAD_DIM, "rotary_dim": HEAD_DIM, "layout": "half", "norm": True, "backward": True,
         "factor": 1.0, "dtype": "bfloat16"},
    ]


def _spread(rng, low, high, step=1):
    """A multiple of ``step`` in [low, high], spread over the logarithm."""

    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high // step * step, max(-(-low // step) * step, round(value / step) * step))


def draw(rng) -> dict:
    kind = rng.choice(["quantize", "forward", "forward", "backward", "weight", "rotary"])
    if kind == "quantize":
        form = rng.choice(["rows", "columns", "both", "weight"])
        return {"kind": kind, "form": form, "rows": _spread(rng, 1, MOST_ROWS), "cols": _spread(rng, 64, FFN, 16),
                "dtype": rng.choice(list(DTYPES))}
    if kind == "rotary":
        head_dim = rng.choice([64, 80, 96, 128, 128, 256])
        heads = rng.choice([8, 16, 24, 32])
        batch = rng.choice([1, 1, 2, 5, 16])
        tokens = _spread(rng, 1, min(8192, 4608 * HEADS * HEAD_DIM // (batch * heads * head_dim)))
        return {"kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": heads // rng.choice([1, 1, 4]),
                "head_dim": head_dim, "rotary_dim": head_dim // rng.choice([1, 1, 2]),
                "layout": rng.choice(["half", "interleaved"]), "norm": rng.random() < 0.5,
                "backward": rng.random() < 0.6, "factor": rng.choice([1.0, 4.0, 8.0]), "dtype": rng.choice(list(DTYPES))}
    in_features, out_features = _spread(rng, 64, MOST_FEATURES, 16), _spread(rng, 64, MOST_FEATURES, 16)
    while in_features * out_features > 2 * FFN * DIM:
        in_features, out_features = _spread(rng, 64, MOST_FEATURES, 16), _spread(rng, 64, MOST_FEATURES, 16)
    most = 4608 * 2 * FFN * DIM // (in_features * out_features)
    case = {"kind": kind, "rows": _spread(rng, 1, min(MOST_ROWS, most)), "in": in_features, "out": out_features,
            "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"])}
    if kind == "weight":
        return {**case, "gradient": rng.choice(["float32", "bfloat16"])}
    case["scales"] = rng.choice(["power", "float32"])
    return {**case, "bias": rng.random() < 0.5} if kind == "forward" else case


# ---- inputs ------------------------------------------------------------------------------------


def _power(exponent):
    """2**exponent, exact (a library's power or exponential of 2 need not be), for -126 <= exponent <= 127."""

    return ((exponent.to(torch.int32) + 127) << 23).view(torch.float32)


def _activations(rows, cols, dtype, g):
    """Rows with a few strong channels, as the outputs of a norm and a modulation have them."""

    gain = torch.exp(0.7 * torch.randn(cols, device="cuda", generator=g))
    return (torch.randn(rows, cols, device="cuda", generator=g) * gain).to(dtype)


def _weight(out_features, in_features, scales, g):
    """A block-scaled weight as a checkpoint or a loader leaves it: (e4m3 values, one scale a block)."""

    weight = 0.02 * torch.randn(out_features, in_features, device="cuda", generator=g)
    rows, cols = -(-out_features // GROUP), -(-in_features // GROUP)
    blocks = torch.zeros(rows * GROUP, cols * GROUP, device="cuda")
    blocks[:out_features, :in_features] = weight
    blocks = blocks.view(rows, GROUP, cols, GROUP)
    peak = blocks.abs().amax((1, 3))
    if scales == "float32":
        scale = peak / 448.0
    else:
        mantissa, exponent = torch.frexp(peak)
        scale = _power(exponent - torch.where(mantissa <= 0.875, 9, 8))
    values = (blocks / scale[:, None, :, None]).view(rows * GROUP, cols * GROUP)[:out_features, :in_features]
    values = values.clamp(-448.0, 448.0).contiguous().to(torch.float8_e4m3fn)
    return values, scale if scales == "float32" else scale.to(torch.float8_e8m0fnu)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    state = {"case": case}
    if kind == "quantize":
        state["x"] = _activations(case["rows"], case["cols"], dtype, g)
        if case["form"] == "weight":
            state["x"] = state["x"] * 0.02
        return state
    if kind == "rotary":
        batch, tokens, heads, kv, head = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
        # queries, keys and values of one fused projection: the queries and keys are views of its output
        fused = torch.randn(batch, tokens, (heads + 2 * kv) * head, device="cuda", generator=g).to(dtype)
        state["q"] = fused[..., : heads * head].unflatten(-1, (heads, head))
        state["k"] = fused[..., heads * head : (heads + kv) * head].unflatten(-1, (kv, head))
        # positions: a stretch from a random start for every sequence (sampling resumes anywhere)
        start = torch.randint(0, int(16384 * case["factor"]), (batch, 1, 1), device="cuda", generator=g)
        state["coordinates"] = (start + torch.arange(tokens, device="cuda")[None, :, None]).float()
        half = case["rotary_dim"] // 2
        exponent = torch.arange(half, device="cuda", dtype=torch.float64) / half
        state["bands"] = (1.0 / (10000.0**exponent * case["factor"])).float()
        state["amplitude"] = 0.1 * math.log(case["factor"]) + 1.0
        state["q_weight"] = state["k_weight"] = None
        if case["norm"]:
            state["q_weight"] = 1.0 + 0.1 * torch.randn(head, device="cuda", generator=g)
            state["k_weight"] = 1.0 + 0.1 * torch.randn(head, device="cuda", generator=g)
        if case["backward"]:
            state["grad_q"] = torch.randn(batch, tokens, heads, head, device="cuda", generator=g).to(dtype)
            state["grad_k"] = torch.randn(batch, tokens, kv, head, device="cuda", generator=g).to(dtype)
        return state
    if kind != "weight":
        state["weight"], state["scale"] = _weight(case["out"], case["in"], case["scales"], g)
    if kind != "backward":
        state["tokens"] = _activations(case["rows"], case["in"], dtype, g)
    if kind != "forward":
        state["gradient"] = 1e-4 * torch.randn(case["rows"], case["out"], device="cuda", generator=g)
        state["gradient"] = state["gradient"].to(dtype)
    state["bias"] = None
    if case.get("bias"):
        state["bias"] = torch.randn(case["out"], device="cuda", generator=g).to(dtype)
    return state


# ---- one pass ----------------------------------------------------------------------------------


def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    fp8, rotary = _framework()
    case = state["case"]
    kind = case["kind"]
    if kind == "quantize":
        x, form = state["x"], case["form"]
        if form == "both":
            rows, columns = fp8.fp8_quantize_both(x)
            return {"rows": fp8.fp8_decode(*rows, dtype=x.dtype),
                    "columns": fp8.fp8_decode(*columns, dtype=x.dtype, cols=x.shape[0])}
        if form == "columns":
            return {"columns": fp8.fp8_decode(*fp8.fp8_quantize_columns(x), dtype=x.dtype, cols=x.shape[0])}
        quantize = fp8.fp8_quantize_rows if form == "rows" else fp8.fp8_quantize_weight
        return {form: fp8.fp8_decode(*quantize(x), dtype=x.dtype)}
    if kind == "forward":
        return fp8.fp8_linear_forward(state["tokens"], state["weight"], state["scale"], state["bias"])
    if kind == "backward":
        return fp8.fp8_linear_backward(state["gradient"], state["weight"], state["scale"])
    if kind == "weight":
        return fp8.fp8_weight_gradient(state["gradient"], state["tokens"], dtype=DTYPES[case["gradient"]])
    table = rotary.rotary_table(state["coordinates"], state["bands"], amplitude=state["amplitude"])
    how = {"layout": case["layout"], "q_weight": state["q_weight"], "k_weight": state["k_weight"]}
    q, k = rotary.rotary_forward(state["q"], state["k"], table, **how)
    if not case["backward"]:
        return [q, k]
    return [q, k, *rotary.rotary_backward(state["grad_q"], state["grad_k"], table, state["q"], state["k"], **how)]


def _padded(x):
    rows, cols = x.shape
    return torch.nn.functional.pad(x, (0, -cols % GROUP)).view(rows, -1, GROUP)


def _read_back(x):
    """Rows in 32 bits to the values that 8 bits keep of them: e4m3 under a power of two for each 128."""

    groups = _padded(x.float())
    mantissa, exponent = torch.frexp(groups.abs().amax(-1, keepdim=True))
    exponent = (exponent - torch.where(mantissa <= 0.875, 9, 8)).clamp(min=-126)
    values = (groups * _power(-exponent)).to(torch.float8_e4m3fn).float()
    return (values * _power(exponent)).flatten(1)[:, : x.shape[1]]


def _weight_back(x):
    rows, cols = x.shape
    blocks = torch.nn.functional.pad(x.float(), (0, -cols % GROUP, 0, -rows % GROUP))
    across = blocks.shape[1] // GROUP
    lines = blocks.view(-1, GROUP, across, GROUP).transpose(1, 2).reshape(-1, GROUP * GROUP)
    mantissa, exponent = torch.frexp(lines.abs().amax(-1, keepdim=True))
    exponent = (exponent - torch.where(mantissa <= 0.875, 9, 8)).clamp(min=-126)
    lines = (lines * _power(-exponent)).to(torch.float8_e4m3fn).float() * _power(exponent)
    return lines.view(-1, across, GROUP, GROUP).transpose(1, 2).reshape(blocks.shape)[:rows, :cols]


def _decoded(weight, scale):
    scale = scale.float().repeat_interleave(GROUP, 0)[: weight.shape[0]]
    return weight.float() * scale.repeat_interleave(GROUP, 1)[:, : weight.shape[1]]


def _rotate(x, sin, cos, layout, rotary):
    """The first ``rotary`` values of each head turned by the table's angles."""

    turned, rest = x[..., :rotary], x[..., rotary:]
    if layout == "half":
        first, second = turned.chunk(2, -1)
        turned = torch.cat((first * cos - second * sin, second * cos + first * sin), -1)
    else:
        first, second = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((first * cos - second * sin, second * cos + first * sin), -1).flatten(-2)
    return torch.cat((turned, rest), -1)


def _rotary_plain(x, weight, sin, cos, grad, layout, rotary):
    x = x.float()
    rms = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) if weight is not None else None
    normed = x * rms * weight if weight is not None else x
    out = _rotate(normed, sin, cos, layout, rotary)
    if grad is None:
        return out, None, None
    back = _rotate(grad.float(), -sin, cos, layout, rotary)
    if weight is None:
        return out, back, None
    unit = x * rms
    inner = back * weight
    back_x = rms * (inner - unit * (inner * unit).mean(-1, keepdim=True))
    return out, back_x, (back * unit).sum((0, 1, 2))


def _run_plain(state):
    case = state["case"]
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "quantize":
        x, form = state["x"], case["form"]
        out = {}
        if form in ("rows", "both"):
            out["rows"] = _read_back(x).to(dtype)
        if form in ("columns", "both"):
            out["columns"] = _read_back(x.t()).to(dtype)
        if form == "weight":
            out["weight"] = _weight_back(x).to(dtype)
        return out
    if kind == "forward":
        y = _read_back(state["tokens"]) @ _decoded(state["weight"], state["scale"]).t()
        return (y if state["bias"] is None else y + state["bias"].float()).to(dtype)
    if kind == "backward":
        return (_read_back(state["gradient"]) @ _decoded(state["weight"], state["scale"])).to(dtype)
    if kind == "weight":
        product = _read_back(state["gradient"].t()) @ _read_back(state["tokens"].t()).t()
        return product.to(DTYPES[case["gradient"]])
    phase = state["coordinates"] * state["bands"]
    sin = (phase.sin() * state["amplitude"]).unsqueeze(-2)
    cos = (phase.cos() * state["amplitude"]).unsqueeze(-2)
    outs, backs, sums = [], [], []
    for name in ("q", "k"):
        out, back, total = _rotary_plain(state[name], state[name + "_weight"], sin, cos, state.get("grad_" + name),
                                         case["layout"], case["rotary_dim"])
        outs.append(out.to(dtype))
        if back is not None:
            backs.append(back.to(dtype))
            sums.append(total)
    return outs + backs + sums


# ---- what a pass cannot do without --------------------------------------------------------------


def work(case: dict) -> dict:
    kind, size = case["kind"], DTYPES[case["dtype"]].itemsize
    if kind == "quantize":
        count = case["rows"] * case["cols"]
        ways = 2 if case["form"] == "both" else 1
        # the matrix read, its 8-bit values written and read back, and the decoded matrix written
        return {"bytes": count * (size + ways * (2 + size)), "flops": ways * 3 * count}
    if kind == "rotary":
        q = case["batch"] * case["tokens"] * case["head_dim"] * (case["heads"] + case["kv_heads"])
        moved = q * size * (5 if case["norm"] and case["backward"] else 4 if case["backward"] else 2)
        table = case["batch"] * case["tokens"] * case["rotary_dim"] * 4
        return {"bytes": moved + table, "flops": q * (12 if case["backward"] else 3)}
    rows, features, weight = case["rows"], (case["in"], case["out"]), case["in"] * case["out"]
    flops = 2 * rows * weight
    if kind == "weight":
        return {"bytes": rows * sum(features) * size + weight * DTYPES[case["gradient"]].itemsize, "flops": flops}
    scales = -(-case["in"] // GROUP) * -(-case["out"] // GROUP) * (4 if case["scales"] == "float32" else 1)
    bias = case["out"] * size if case.get("bias") else 0
    return {"bytes": rows * sum(features) * size + weight + scales + bias, "flops": flops}


# ---- the definition in 64 bits ------------------------------------------------------------------


def _exact_groups(x):
    """What 8 bits keep of the last dimension's groups of 128, from the definition of e4m3: four significant
    bits down to 2**-6, steps of 2**-9 below, ties to the even step, under the smallest power of two (from
    2**-126 on) that brings the group within 448."""

    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    whole = x.shape[-1] // GROUP * GROUP
    for piece, to in ((x[..., :whole].unflatten(-1, (-1, GROUP)) if whole else None, slice(0, whole)),
                      (x[..., None, whole:] if whole < x.shape[-1] else None, slice(whole, None))):
        if piece is not None:
            out[..., to] = _exact_block(piece.double(), (-1,)).flatten(-2)
    return out


def _exact_block(x, dims):
    powers = torch.tensor([2.0**i for i in range(-200, 200)], dtype=torch.float64, device=x.device)
    peak = x.abs().amax(dims, keepdim=True).unsqueeze(-1)
    index = 74 + torch.arange(247, device=x.device)  # 2**-126 to 2**120
    fits = peak <= 448.0 * powers[index]
    power = powers[index[fits.to(torch.uint8).argmax(-1)]]
    v = x / power
    # the step of a value between 2**i and 2**(i + 1) is 2**(i - 3), and 2**-9 below 2**-6
    step = torch.full_like(v, 2.0**-9)
    for i in range(-6, 9):
        step[v.abs() >= 2.0**i] = 2.0 ** (i - 3)
    return torch.round(v / step) * step * power


def _exact_weight(weight, scale):
    out = weight.to(torch.float64)
    for i in range(scale.shape[0]):
        rows = slice(i * GROUP, (i + 1) * GROUP)
        out[rows] *= scale[i].double().repeat_interleave(GROUP)[: weight.shape[1]]
    return out


def _exact_rotary(x, weight, phase, amplitude, grad, layout, rotary):
    x = x.double()
    head = x.shape[-1]
    # the rotation as a complex product on pairs
    index = torch.arange(rotary, device=x.device)
    pairs = index.view(2, -1).t() if layout == "half" else index.view(-1, 2)
    spin = torch.polar(torch.full_like(phase, amplitude), phase).unsqueeze(-2)

    def turn(v, by):
        out = v.clone()
        z = torch.complex(v[..., pairs[:, 0]], v[..., pairs[:, 1]]) * by
        out[..., pairs[:, 0]], out[..., pairs[:, 1]] = z.real, z.imag
        return out

    if weight is None:
        return turn(x, spin), None if grad is None else turn(grad.double(), spin.conj()), None
    length = (x.pow(2).sum(-1, keepdim=True) / head + 1e-6).sqrt()
    unit = x / length
    out = turn(unit * weight.double(), spin)
    if grad is None:
        return out, None, None
    back = turn(grad.double(), spin.conj())
    scaled = back * weight.double()
    along = (scaled * x).sum(-1, keepdim=True) / (head * length.pow(3))
    return out, scaled / length - x * along, (back * unit).flatten(0, 2).sum(0)


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        x, form = state["x"], case["form"]
        out = {}
        if form in ("rows", "both"):
            out["rows"] = _exact_groups(x)
        if form in ("columns", "both"):
            out["columns"] = _exact_groups(x.t())
        if form == "weight":
            out["weight"] = torch.empty(x.shape, dtype=torch.float64, device=x.device)
            for i in range(0, x.shape[0], GROUP):
                for j in range(0, x.shape[1], GROUP):
                    block = (slice(i, i + GROUP), slice(j, j + GROUP))
                    out["weight"][block] = _exact_block(x[block].double(), (0, 1))
        return out
    if kind == "forward":
        y = _exact_groups(state["tokens"]) @ _exact_weight(state["weight"], state["scale"]).t()
        return y if state["bias"] is None else y + state["bias"].double()
    if kind == "backward":
        return _exact_groups(state["gradient"]) @ _exact_weight(state["weight"], state["scale"])
    if kind == "weight":
        return _exact_groups(state["gradient"].t()) @ _exact_groups(state["tokens"].t()).t()
    # an angle is the 32-bit product of a coordinate and a band, as positions are defined
    phase = (state["coordinates"] * state["bands"]).double()
    sides = [_exact_rotary(state[n], state[n + "_weight"], phase, state["amplitude"], state.get("grad_" + n),
                           case["layout"], case["rotary_dim"]) for n in ("q", "k")]
    if not case["backward"]:
        return [s[0] for s in sides]
    return [s[i] for i in range(3) for s in sides]
