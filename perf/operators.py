"""Cases of the 8-bit feed-forward operators: RMS norm with the residual's addition (for training, and with 8-bit rows
for serving), the 8-bit matrix product with token and channel scales, and SwiGLU with 8-bit activation checkpoints (for
training) or 8-bit rows (for serving).

`run` computes an operator's plain form in elementary torch operations, or, with `own` set, makes the framework's calls;
`exact` gives the same outputs from the definitions in 64 bits."""

import math
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-6
GROUP = 128  # channels of a gate or value row that share one checkpoint scale
PACKAGE = str(Path(__file__).resolve().parent.parent / "jittor-flow2surf_b200")
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # one norm of the trunk's residual stream in training: 64 patches x 1,024 points, width 192
        {"name": "norm_train_trunk", "op": "norm_train", "rows": 65536, "width": 192, "type": "bfloat16", "residual": True},
        # a ragged batch of odd width in single precision
        {"name": "norm_train_odd", "op": "norm_train", "rows": 4099, "width": 1531, "type": "float32", "residual": True},
        # one token of a generic model width, where latency counts
        {"name": "norm_int8_token", "op": "norm_int8", "rows": 1, "width": 4096, "type": "float16", "residual": True},
        # a long prompt of the same width
        {"name": "norm_int8_prompt", "op": "norm_int8", "rows": 32768, "width": 4096, "type": "bfloat16", "residual": True},
        # one token through a square projection: the weights' bytes
        {"name": "linear_token", "op": "linear_int8", "rows": 1, "width": 4096, "cols": 4096, "type": "bfloat16", "quantize": False, "bias": False},
        # a few tokens in flight, odd sizes, rows that come in 16 bits, single-precision logits
        {"name": "linear_few_odd", "op": "linear_int8", "rows": 24, "width": 2049, "cols": 6151, "type": "float32", "quantize": True, "bias": True},
        # the trunk's first feed-forward projection at its training batch
        {"name": "linear_trunk", "op": "linear_int8", "rows": 65536, "width": 192, "cols": 1536, "type": "float16", "quantize": False, "bias": True},
        # a large square product: the arithmetic
        {"name": "linear_large", "op": "linear_int8", "rows": 8192, "width": 8192, "cols": 8192, "type": "bfloat16", "quantize": True, "bias": False},
        # a feed-forward activation at the trunk's training batch
        {"name": "swiglu_train_trunk", "op": "swiglu_train", "rows": 65536, "hidden": 1024, "type": "bfloat16"},
        # an odd hidden width (a last group of 91 channels) in single precision
        {"name": "swiglu_train_odd", "op": "swiglu_train", "rows": 2053, "hidden": 1371, "type": "float32"},
        # a few tokens of a served batch
        {"name": "swiglu_int8_tokens", "op": "swiglu_int8", "rows": 8, "hidden": 6144, "type": "bfloat16"},
        # a long prompt
        {"name": "swiglu_int8_prompt", "op": "swiglu_int8", "rows": 16384, "hidden": 4096, "type": "float16"},
    ]


def _size(rng, low, high):
    """A size of [low, high], spread over its logarithm: half of them as they fall, half a multiple of 64 where that is in the range."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and n >= 64:
        n -= n % 64
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["norm_train", "norm_int8", "linear_int8", "swiglu_train", "swiglu_int8"])
    rows = _size(rng, 1, 65536)
    if op == "linear_int8":
        width, cols = _size(rng, 32, 8192), _size(rng, 32, 8192)
        rows = max(1, min(rows, 8192**3 // (width * cols), 2**26 // cols, 2**26 // width))
        return {"op": op, "rows": rows, "width": width, "cols": cols, "type": rng.choice(list(TYPES)), "quantize": rng.random() < 0.5, "bias": rng.random() < 0.5}
    if op in ("norm_train", "norm_int8"):
        width = _size(rng, 16, 8192)
        most = 2**27 if op == "norm_int8" else 65536 * 192
        return {"op": op, "rows": max(1, min(rows, most // width)), "width": width, "type": rng.choice(list(TYPES)), "residual": rng.random() < 0.75}
    hidden = _size(rng, 16, 8192)
    rows = max(1, min(rows, 2**25 // hidden))
    # a served row of 8 bits comes from a 16-bit projection
    return {"op": op, "rows": rows, "hidden": hidden, "type": rng.choice(list(TYPES) if op == "swiglu_train" else ["bfloat16", "float16"])}


def _pitched(values):
    """An int8 matrix whose rows start 16-byte aligned, as the framework's quantiser lays them out."""
    rows, width = values.shape
    held = torch.zeros(rows, -(-width // 16) * 16, dtype=torch.int8, device=values.device)
    held[:, :width] = values
    return held[:, :width]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]
    rows = case["rows"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def eighth(*shape):  # 8-bit values of a normal row or channel, whose largest magnitude is about 4.5 sigma
        return _pitched((normal(*shape) * 28).round_().clamp_(-127, 127).to(torch.int8))

    state = {"op": case["op"], "dtype": dtype}
    if case["op"] in ("norm_train", "norm_int8"):
        train = case["op"] == "norm_train"
        width = case["width"]
        # a residual stream has a few channels of much larger magnitude than the rest
        loud = 1 + 15 * (torch.rand(width, generator=g, device="cuda") < 0.02)
        state["x"] = normal(rows, width).to(dtype).requires_grad_(train)
        state["residual"] = (normal(rows, width) * loud).to(dtype).requires_grad_(train) if case["residual"] else None
        state["weight"] = (1 + 0.2 * normal(width)).to(dtype).requires_grad_(train)
        if train:
            state["dy"] = normal(rows, width).to(dtype)
            state["dstream"] = normal(rows, width).to(dtype) if case["residual"] else None
    elif case["op"] == "linear_int8":
        width, cols = case["width"], case["cols"]
        if case["quantize"]:
            state["x"] = normal(rows, width).to(dtype)
        else:
            state["x8"], state["x_scale"] = eighth(rows, width), (0.5 + torch.rand(rows, generator=g, device="cuda")) / 28
        state["w8"], state["w_scale"] = eighth(cols, width), (0.5 + torch.rand(cols, generator=g, device="cuda")) / (28 * width**0.5)
        state["bias"] = normal(cols).to(dtype) if case["bias"] else None
    else:
        train = case["op"] == "swiglu_train"
        state["projected"] = (1.5 * normal(rows, 2 * case["hidden"])).to(dtype).requires_grad_(train)
        if train:
            state["dy"] = normal(rows, case["hidden"]).to(dtype)
    return state


# ---- the plain forms: 32 bits, the 8-bit rounding (next to its borders) in 64 ----


def _eight_bits(values):
    """Whole numbers of [-127, 127] for each row of 64-bit values and the row's largest magnitude."""
    largest = values.abs().amax(-1, keepdim=True)
    return torch.where(largest > 0, values * 127 / largest, 0).round().float(), largest


def _norm_plain(state):
    x, residual, dtype = state["x"].detach(), state["residual"], state["dtype"]
    weight = state["weight"].detach().float()
    stream = x if residual is None else (x.float() + residual.detach().float()).to(dtype)
    s = stream.float()
    return s, torch.rsqrt(s.square().mean(-1, keepdim=True) + EPS), weight, stream


def _norm_train_plain(state):
    s, rstd, weight, stream = _norm_plain(state)
    dtype = state["dtype"]
    dy = state["dy"].float()
    normed = s * rstd
    y = (normed * weight).to(dtype)
    u = dy * weight
    grad = rstd * (u - normed * (u * normed).mean(-1, keepdim=True))
    dweight = (dy * normed).sum(0).to(dtype)
    if state["residual"] is None:
        return {"y": y, "dx": grad.to(dtype), "dweight": dweight}
    grad = (grad + state["dstream"].float()).to(dtype)
    return {"y": y, "stream": stream, "dx": grad, "dresidual": grad, "dweight": dweight}


def _norm_int8_plain(state):
    s, rstd, weight, stream = _norm_plain(state)
    q, largest = _eight_bits(s.double() * weight.double())
    y = (q * (largest / 127 * rstd).float()).to(state["dtype"])
    return {"y": y} if state["residual"] is None else {"y": y, "stream": stream}


def _linear_plain(state):
    if "x" in state:
        x, largest = _eight_bits(state["x"].double())
        scale = (largest / 127).float()
    else:
        x, scale = state["x8"].float(), state["x_scale"][:, None]
    y = x @ state["w8"].float().T * scale * state["w_scale"]
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return {"y": y.to(state["dtype"])}


def _kept(values):
    """What an 8-bit checkpoint of (rows, hidden) values stands for."""
    rows, hidden = values.shape
    groups = -(-hidden // GROUP)
    held = values.new_zeros(rows, groups * GROUP, dtype=torch.float64)
    held[:, :hidden] = values
    q, largest = _eight_bits(held.view(rows, groups, GROUP))
    return (q * (largest / 127).float()).view(rows, groups * GROUP)[:, :hidden]


def _swiglu_train_plain(state):
    projected, dtype = state["projected"].detach(), state["dtype"]
    gate, value = projected.chunk(2, dim=-1)
    y = (gate.float() * torch.sigmoid(gate.float()) * value.float()).to(dtype)
    gate, value, dy = _kept(gate), _kept(value), state["dy"].float()
    sigma = torch.sigmoid(gate)
    dgate = dy * value * sigma * (1 + gate * (1 - sigma))
    dvalue = dy * gate * sigma
    return {"y": y, "dprojected": torch.cat([dgate, dvalue], dim=-1).to(dtype)}


def _swiglu_int8_plain(state):
    gate, value = state["projected"].float().chunk(2, dim=-1)
    q, largest = _eight_bits((gate * torch.sigmoid(gate) * value).double())
    return {"y": (q * (largest / 127).float()).to(state["dtype"])}


PLAIN = {
    "norm_train": _norm_train_plain,
    "norm_int8": _norm_int8_plain,
    "linear_int8": _linear_plain,
    "swiglu_train": _swiglu_train_plain,
    "swiglu_int8": _swiglu_int8_plain,
}


# ---- the framework's calls ----


def _framework():
    """The package; a user's program has it imported from the start."""
    if "flow2surf_b200" not in sys.modules and PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import flow2surf_b200

    return flow2surf_b200


def _norm_train_own(f2s, state):
    x, residual, weight = state["x"], state["residual"], state["weight"]
    y, stream = f2s.add_rms_norm(x, weight, residual, eps=EPS)
    if residual is None:
        dx, dweight = torch.autograd.grad(y, (x, weight), state["dy"])
        return {"y": y, "dx": dx, "dweight": dweight}
    dx, dresidual, dweight = torch.autograd.grad((y, stream), (x, residual, weight), (state["dy"], state["dstream"]))
    return {"y": y, "stream": stream, "dx": dx, "dresidual": dresidual, "dweight": dweight}


def _norm_int8_own(f2s, state):
    rows8, stream = f2s.add_rms_norm_int8(state["x"], state["weight"], state["residual"], eps=EPS)
    y = rows8.dequantize(state["dtype"])
    return {"y": y} if state["residual"] is None else {"y": y, "stream": stream}


def _linear_own(f2s, state):
    rows8 = f2s.quantize_rows(state["x"]) if "x" in state else f2s.Int8Rows(state["x8"], state["x_scale"])
    return {"y": f2s.linear_int8(rows8, f2s.Int8Rows(state["w8"], state["w_scale"]), state["bias"], dtype=state["dtype"])}


def _swiglu_train_own(f2s, state):
    y = f2s.swiglu(state["projected"], checkpoint="int8")
    return {"y": y, "dprojected": torch.autograd.grad(y, state["projected"], state["dy"])[0]}


def _swiglu_int8_own(f2s, state):
    return {"y": f2s.swiglu_int8(state["projected"]).dequantize(state["dtype"])}


OWN = {
    "norm_train": _norm_train_own,
    "norm_int8": _norm_int8_own,
    "linear_int8": _linear_own,
    "swiglu_train": _swiglu_train_own,
    "swiglu_int8": _swiglu_int8_own,
}


def run(state):
    if own:
        return OWN[state["op"]](_framework(), state)
    with torch.no_grad():
        return PLAIN[state["op"]](state)


def work(case):
    rows, size = case["rows"], TYPES[case["type"]].itemsize
    if case["op"] == "linear_int8":
        width, cols = case["width"], case["cols"]
        held = rows * width * (size if case["quantize"] else 1) + (0 if case["quantize"] else 4 * rows)
        return {"bytes": held + cols * (width + 4 + (size if case["bias"] else 0)) + rows * cols * size, "flops": 2 * rows * width * cols}
    if case["op"] == "norm_train":  # x, dy to y, dx; with a residual also r, dstream to the stream
        return {"bytes": rows * case["width"] * size * (7 if case["residual"] else 4), "flops": 14 * rows * case["width"]}
    if case["op"] == "norm_int8":
        return {"bytes": rows * case["width"] * size * (4 if case["residual"] else 2), "flops": 8 * rows * case["width"]}
    if case["op"] == "swiglu_train":  # gate, value, dy to y, dgate, dvalue
        return {"bytes": rows * case["hidden"] * size * 6, "flops": 24 * rows * case["hidden"]}
    return {"bytes": rows * case["hidden"] * size * 3, "flops": 10 * rows * case["hidden"]}


# ---- the definitions in 64 bits ----


def _nearest_whole(values, largest):
    """The whole numbers nearest to 127 v / m, the even one at a tie, by comparing with the halves on both sides."""
    below = torch.floor(127 * values / torch.where(largest > 0, largest, 1))
    twice = 254 * values - (2 * below + 1) * largest
    up = (twice > 0) | ((twice == 0) & (below.remainder(2) == 1))
    return torch.where(largest > 0, below + up, 0)


def exact(case, seed):
    state = prepare(case, seed)
    wide = {k: v.detach().double() for k, v in state.items() if isinstance(v, torch.Tensor)}
    with torch.no_grad():
        if case["op"] in ("norm_train", "norm_int8"):
            total = wide["x"]
            if case["residual"]:
                total = total + wide["residual"]
            stream = total.float().to(state["dtype"]).double()  # the norm reads the stream that is stored
            power = torch.einsum("rc,rc->r", stream, stream)[:, None] / case["width"] + EPS
            got = {"stream": total} if case["residual"] else {}
            if case["op"] == "norm_int8":
                weighted = stream * wide["weight"]
                largest = torch.maximum(weighted.amax(-1), -weighted.amin(-1))[:, None]
                got["y"] = _nearest_whole(weighted, largest) * largest / (127 * power.sqrt())
                return got
            got["y"] = stream * wide["weight"] / power.sqrt()
            towards = wide["dy"] * wide["weight"]
            along = torch.einsum("rc,rc->r", towards, stream)[:, None] / (case["width"] * power)
            got["dx"] = (towards - along * stream) / power.sqrt()
            got["dweight"] = torch.einsum("rc,rc->c", wide["dy"], stream / power.sqrt())
            if case["residual"]:
                got["dx"] = got["dx"] + wide["dstream"]
                got["dresidual"] = got["dx"]
            return got
        if case["op"] == "linear_int8":
            if case["quantize"]:
                largest = wide["x"].abs().max(-1).values[:, None]
                x = _nearest_whole(wide["x"], largest) * largest / 127
            else:
                x = wide["x8"] * wide["x_scale"][:, None]
            y = torch.einsum("rk,nk->rn", x, wide["w8"] * wide["w_scale"][:, None])
            return {"y": y if state["bias"] is None else y + wide["bias"]}
        hidden = case["hidden"]
        gate, value = wide["projected"][:, :hidden], wide["projected"][:, hidden:]
        product = gate * value / (1 + torch.exp(-gate))
        if case["op"] == "swiglu_int8":
            largest = product.abs().max(-1).values[:, None]
            return {"y": _nearest_whole(product, largest) * largest / 127}
        kept = wide["projected"].clone()
        for half in (kept[:, :hidden], kept[:, hidden:]):
            for first in range(0, hidden, GROUP):
                part = half[:, first : first + GROUP]
                largest = part.abs().max(-1).values[:, None]
                part.copy_(_nearest_whole(part, largest) * largest / 127)
        gate, value = kept[:, :hidden], kept[:, hidden:]
        slope = 1 / (1 + torch.exp(-gate))
        down = wide["dy"] * gate * slope
        return {"y": product, "dprojected": torch.cat([wide["dy"] * value * (slope + gate * slope * (1 - slope)), down], dim=1)}
