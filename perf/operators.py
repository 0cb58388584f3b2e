"""The operators of layers served in 8-bit integers, as cases that can be timed and compared.

A layer in 8 bits is: the norm of the stream with int8 rows as its output (``norm``), products of int8 rows with int8 weights
(``linear``), the gated product of a feed-forward (``gated``), and the rounding of an activation or a weight to int8 rows
(``quantize``).  A row of int8 values comes with one float32 scale and stands for values times scale; weights are such rows
too, one per output feature.  Sizes are the layer sizes of Qwen2.5-0.5B, 1.5B and 7B and odd ones between them.

int8 results are returned as the values that they stand for, in bfloat16, beside their scales.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = torch.device("cuda:0")
BF16, F32, F64, I8 = torch.bfloat16, torch.float32, torch.float64, torch.int8
TYPES = {"bf16": BF16, "f32": F32}
EPS = 1e-6
RUN = 64  # gate and up rows of a stacked weight alternate in runs of this many


def listed() -> list[dict]:
    return [
        # attention's output of one decoded token of a small model, in front of the output projection: latency alone
        dict(name="quantize_1_row_of_896", kind="quantize", rows=1, width=896, type="bf16", stride=896),
        # the hidden vectors of a prompt portion at the 7B sizes, in front of the down projection
        dict(name="quantize_2048_rows_of_18944", kind="quantize", rows=2048, width=18944, type="bf16", stride=18944),
        # float32 rows of odd length that stand in a wider tensor (the 32-bit path; a slice of a stacked projection)
        dict(name="quantize_1531_strided_f32", kind="quantize", rows=1531, width=2051, type="f32", stride=2304),
        # between two layers of a decode step with 8 requests
        dict(name="norm_8_rows_of_3584", kind="norm", rows=8, width=3584, type="bf16", weight="bf16"),
        # between two layers of a long prompt portion
        dict(name="norm_4096_rows_of_3584", kind="norm", rows=4096, width=3584, type="bf16", weight="bf16"),
        # odd everything: a ragged portion, float32 branch outputs, a width off every vector size
        dict(name="norm_777_rows_of_1537_f32", kind="norm", rows=777, width=1537, type="f32", weight="f32"),
        # q/k/v of one decoded token of a small model: the smallest product, with its bias
        dict(name="linear_1x896x1152", kind="linear", rows=1, width=896, features=1152, bias=True, type="bf16"),
        # the down projection of a decode step with 16 requests: the weights' bytes are the work
        dict(name="linear_16x18944x3584", kind="linear", rows=16, width=18944, features=3584, bias=False, type="bf16"),
        # requests that decode beside a short portion, odd sizes and float32 outputs: between the two regimes
        dict(name="linear_203x3581x4613_f32", kind="linear", rows=203, width=3581, features=4613, bias=True, type="f32"),
        # q/k/v of a long prompt portion: the tensor cores are the work
        dict(name="linear_2047x3584x4608", kind="linear", rows=2047, width=3584, features=4608, bias=True, type="bf16"),
        # gate and up of a decode step with 8 requests
        dict(name="gated_8x3584x18944", kind="gated", rows=8, width=3584, features=18944, bias=False, type="bf16"),
        # gate and up of a long prompt portion
        dict(name="gated_4099x3584x18944", kind="gated", rows=4099, width=3584, features=18944, bias=False, type="bf16"),
    ]


def _log(rng, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    kind = rng.choice(["quantize", "norm", "linear", "linear", "linear", "gated"])
    rows = _log(rng, 1, 4096)
    if kind == "quantize":
        width = rng.choice([896, 1536, 3584, 4864, 8960, 18944, _log(rng, 17, 12000)])
        return dict(kind=kind, rows=rows, width=width, type=rng.choice(["bf16", "bf16", "f32"]), stride=width + rng.choice([0, 0, 8, 77]))
    if kind == "norm":
        width = rng.choice([896, 1536, 3584, 3584, _log(rng, 17, 8192)])
        return dict(kind=kind, rows=rows, width=width, type=rng.choice(["bf16", "bf16", "f32"]), weight=rng.choice(["bf16", "f32"]))
    if kind == "gated":
        width, features = rng.choice([(896, 4864), (1536, 8960), (3584, 18944), (_log(rng, 33, 4000), RUN * _log(rng, 1, 150))])
        return dict(kind=kind, rows=rows, width=width, features=features, bias=rng.random() < 0.25, type=rng.choice(["bf16", "bf16", "f32"]))
    width, features = rng.choice([(896, 1152), (896, 896), (4864, 896), (1536, 2048), (8960, 1536), (3584, 4608), (3584, 3584),
                                  (18944, 3584), (_log(rng, 33, 19000), _log(rng, 5, 5000)), (_log(rng, 33, 5000), _log(rng, 5, 19000))])
    return dict(kind=kind, rows=rows, width=width, features=features, bias=rng.random() < 0.5, type=rng.choice(["bf16", "bf16", "f32"]))


# --------------------------------------------------------------------------- inputs

def _generator(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(g: torch.Generator, *shape: int, std: float = 1.0, mean: float = 0.0, dtype: torch.dtype = F32) -> torch.Tensor:
    return torch.empty(shape, dtype=F32, device=DEVICE).normal_(mean, std, generator=g).to(dtype)


def _int8_rows(g: torch.Generator, rows: int, width: int, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """Normal values in int8 (every row's largest near 127) and scales that differ by row; rows start on 16 bytes."""
    store = torch.zeros((rows, -(-width // 16) * 16), dtype=I8, device=DEVICE)
    store[:, :width] = _normal(g, rows, width, std=33.0).round_().clamp_(-127, 127).to(I8)
    return store[:, :width], scale * _normal(g, rows, std=0.3).exp()


def prepare(case: dict, seed: int) -> dict:
    g = _generator(seed)
    kind, rows, width, dtype = case["kind"], case["rows"], case["width"], TYPES[case["type"]]
    if kind == "quantize":
        x = _normal(g, rows, case["stride"], dtype=dtype)
        x *= _normal(g, rows, 1, std=0.5).exp().to(dtype)  # tokens differ in size
        if rows > 4:
            x[rows // 2] = 0  # a row of padding
        return dict(kind=kind, x=x[:, :width])
    if kind == "norm":
        residual = _normal(g, rows, width, std=3.0)
        residual[:, :: max(1, width // 7)] *= 6.0  # a few features of a stream are large in every token
        return dict(kind=kind, residual=residual, delta=_normal(g, rows, width, dtype=dtype), out=torch.empty_like(residual),
                    weight=_normal(g, width, std=0.1, mean=1.0, dtype=TYPES[case["weight"]]))
    features = case["features"] * (2 if kind == "gated" else 1)
    x, x_scale = _int8_rows(g, rows, width, 0.03)
    w, w_scale = _int8_rows(g, features, width, 0.03 / math.sqrt(width))
    bias = _normal(g, features, dtype=BF16) if case["bias"] else None
    return dict(kind=kind, x=x, x_scale=x_scale, w=w, w_scale=w_scale, bias=bias, type=dtype)


# --------------------------------------------------------------------------- the operators

def _plain_int8(v: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of float32 to the int8 values (kept in float32) and their scales."""
    top = v.abs().amax(dim=1, keepdim=True)
    scale = top / torch.full_like(top, 127.0)
    inverse = torch.where(top > 0, torch.full_like(top, 127.0) / top, torch.zeros_like(top))
    return (v * inverse).round(), scale


def _plain(state: dict):
    kind = state["kind"]
    if kind == "quantize":
        q, scale = _plain_int8(state["x"].float())
        return (q * scale).to(BF16), scale[:, 0]
    if kind == "norm":
        stream = state["residual"] + state["delta"].float()
        normed = stream * torch.rsqrt((stream * stream).mean(dim=1, keepdim=True) + EPS) * state["weight"].float()
        q, scale = _plain_int8(normed)
        return stream, (q * scale).to(BF16), scale[:, 0]
    y = (state["x"].float() @ state["w"].float().t()) * state["x_scale"][:, None] * state["w_scale"]
    if state["bias"] is not None:
        y = y + state["bias"].float()
    if kind == "gated":
        runs = y.reshape(y.shape[0], -1, 2, RUN)
        gate, up = runs[:, :, 0].reshape(y.shape[0], -1), runs[:, :, 1].reshape(y.shape[0], -1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    return y.to(state["type"])


def _kernels(state: dict):
    from slipstream_b200 import ops

    kind = state["kind"]
    if kind == "quantize":
        rows = ops.quantize_rows_int8(state["x"])
        return ops.dequantize_rows_int8(rows, BF16), rows.scales
    if kind == "norm":
        rows = ops.add_rmsnorm_int8(state["residual"], state["delta"], state["weight"], EPS, residual_out=state["out"])
        return state["out"], ops.dequantize_rows_int8(rows, BF16), rows.scales
    x, w = ops.Int8Rows(state["x"], state["x_scale"]), ops.Int8Rows(state["w"], state["w_scale"])
    if kind == "gated":
        return ops.gate_up_swiglu_int8(x, w, state["bias"], state["type"])
    return ops.linear_int8(x, w, state["bias"], state["type"])


def run(state: dict):
    return _kernels(state) if own else _plain(state)


# --------------------------------------------------------------------------- what a pass needs, and what is exact

def work(case: dict) -> dict:
    rows, width, size = case["rows"], case["width"], 2 if case["type"] == "bf16" else 4
    if case["kind"] == "quantize":  # the row in; int8, its scale and the values it stands for out
        return {"bytes": rows * (width * (size + 1 + 2) + 4), "flops": 3 * rows * width}
    if case["kind"] == "norm":  # stream and branch in; stream, int8, scale and values out
        return {"bytes": rows * (width * (4 + size + 4 + 1 + 2) + 4) + width * (2 if case["weight"] == "bf16" else 4), "flops": 8 * rows * width}
    features = case["features"]
    stacked = 2 * features if case["kind"] == "gated" else features
    return {"bytes": rows * (width + 4) + stacked * (width + 4 + (2 if case["bias"] else 0)) + rows * features * size,
            "flops": 2 * rows * stacked * width}


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind in ("quantize", "norm"):
        if kind == "quantize":
            first, v = [], state["x"].to(F64)
        else:
            stream = state["residual"].to(F64) + state["delta"].to(F64)
            first = [stream]
            v = stream / (stream.square().sum(dim=1, keepdim=True) / case["width"] + EPS).sqrt() * state["weight"].to(F64)
        scale = v.abs().max(dim=1).values / 127
        steps = torch.where(scale[:, None] > 0, v / scale[:, None], torch.zeros_like(v))
        return (*first, torch.round(steps) * scale[:, None], scale)
    out = torch.matmul(state["x"].to(F64), state["w"].to(F64).mT)
    out = out * torch.outer(state["x_scale"].to(F64), state["w_scale"].to(F64))
    if state["bias"] is not None:
        out = out + state["bias"].to(F64)
    if kind == "linear":
        return out
    feature = torch.arange(case["features"], device=DEVICE)
    at = feature // RUN * (2 * RUN) + feature % RUN
    gate, up = out[:, at], out[:, at + RUN]
    return gate * torch.sigmoid(gate) * up
