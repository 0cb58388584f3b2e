"""The operators of layers served in 8-bit floats and of a model's log probabilities, as cases that can be timed and compared.

A layer in 8-bit floats is: the rounding of a tensor to e4m3 with one float32 scale for each block of 128 (``quantize``: blocks of 128
elements of a row, or of 128 x 128 elements of a weight), the norm of the stream that ends in such rows (``norm``), products of
such rows with such weights (``linear``) and the gated product of a feed-forward (``gated``), which may end in such rows again.
What a model answers with (``logprobs``) is, for each row of logits, the log probability of a given token and its rank, the entropy
of the distribution, and the largest log probabilities with their tokens.  Sizes are the layer sizes and vocabularies of
Qwen2.5-0.5B, 1.5B and 7B and odd ones between them.

8-bit results are returned as the values that they stand for, in bfloat16, beside their scales.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = torch.device("cuda:0")
BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
TYPES = {"bf16": BF16, "f32": F32, "fp8": E4M3}
SIZES = {"bf16": 2, "f32": 4, "fp8": 1}
EPS = 1e-6
BLOCK = 128  # elements that share a scale; gate and up rows of a stacked weight alternate in runs of as many
TOP = 448.0  # the largest e4m3


def listed() -> list[dict]:
    return [
        # an activation of odd width that stands in a wider float32 tensor (a slice of a stacked projection)
        dict(name="quantize_1531_strided_rows_f32", kind="quantize", form="rows", rows=1531, width=2051, type="f32", stride=2304),
        # the gate matrix of a layer at the 7B sizes, as it is bound
        dict(name="quantize_weight_18944x3584", kind="quantize", form="blocks", rows=18944, width=3584, type="bf16", stride=3584),
        # between two layers of a decode step with 8 requests: latency
        dict(name="norm_8_rows_of_3584", kind="norm", rows=8, width=3584, type="bf16", weight="bf16"),
        # between two layers of a long prompt portion
        dict(name="norm_4096_rows_of_3584", kind="norm", rows=4096, width=3584, type="bf16", weight="bf16"),
        # q/k/v of one decoded token of a small model: the smallest product, with its bias
        dict(name="linear_1x896x1152", kind="linear", rows=1, width=896, features=1152, bias=True, type="bf16"),
        # the down projection of a decode step with 16 requests: the weights' bytes are the work
        dict(name="linear_16x18944x3584", kind="linear", rows=16, width=18944, features=3584, bias=False, type="bf16"),
        # a ragged prompt portion, odd sizes everywhere and float32 outputs
        dict(name="linear_2047x3581x4613_f32", kind="linear", rows=2047, width=3581, features=4613, bias=True, type="f32"),
        # gate and up of a decode step with 8 requests, rounded for the down projection
        dict(name="gated_8x3584x18944_fp8", kind="gated", rows=8, width=3584, features=18944, bias=False, type="fp8"),
        # gate and up of a long prompt portion
        dict(name="gated_4099x3584x18944", kind="gated", rows=4099, width=3584, features=18944, bias=False, type="bf16"),
        # one decoded token whose caller asked for alternatives: latency
        dict(name="logprobs_1x151936_top5", kind="logprobs", rows=1, vocabulary=151936, type="f32", top=5, masked=0.0),
        # a decode step of a guided batch over a vocabulary of odd size: most tokens masked, the tokens' own log probabilities alone
        dict(name="logprobs_67x50257_masked", kind="logprobs", rows=67, vocabulary=50257, type="bf16", top=0, masked=0.9),
        # a prompt portion that is scored token by token
        dict(name="logprobs_1024x151936_top20", kind="logprobs", rows=1024, vocabulary=151936, type="f32", top=20, masked=0.0),
    ]


def _log(rng, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    kind = rng.choice(["quantize", "norm", "linear", "linear", "gated", "logprobs", "logprobs"])
    rows = _log(rng, 1, 4096)
    if kind == "quantize":
        width = rng.choice([896, 1536, 3584, 4864, 8960, 18944, _log(rng, 17, 12000)])
        return dict(kind=kind, form=rng.choice(["rows", "rows", "blocks"]), rows=rows, width=width, type=rng.choice(["bf16", "bf16", "f32"]),
                    stride=width + rng.choice([0, 0, 8, 77]))
    if kind == "norm":
        width = rng.choice([896, 1536, 3584, 3584, _log(rng, 17, 8192)])
        return dict(kind=kind, rows=rows, width=width, type=rng.choice(["bf16", "bf16", "f32"]), weight=rng.choice(["bf16", "f32"]))
    if kind == "gated":
        width, features = rng.choice([(896, 4864), (1536, 8960), (3584, 18944), (_log(rng, 33, 3500), _log(rng, 100, 18900))])
        return dict(kind=kind, rows=rows, width=width, features=features, bias=rng.random() < 0.25, type=rng.choice(["bf16", "fp8", "fp8", "f32"]))
    if kind == "logprobs":
        vocabulary = rng.choice([151936, 152064, _log(rng, 1000, 152000)])
        return dict(kind=kind, rows=_log(rng, 1, 1000), vocabulary=vocabulary, type=rng.choice(["f32", "f32", "bf16"]), top=rng.choice([0, 1, 5, 20]),
                    masked=rng.choice([0.0, 0.0, 0.9]))
    width, features = rng.choice([(896, 1152), (896, 896), (4864, 896), (1536, 2048), (8960, 1536), (3584, 4608), (3584, 3584),
                                  (18944, 3584), (_log(rng, 33, 19000), _log(rng, 5, 5000)), (_log(rng, 33, 5000), _log(rng, 5, 19000))])
    return dict(kind=kind, rows=rows, width=width, features=features, bias=rng.random() < 0.5, type=rng.choice(["bf16", "bf16", "f32"]))


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


# --------------------------------------------------------------------------- inputs

def _generator(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(g: torch.Generator, *shape: int, std: float = 1.0, mean: float = 0.0, dtype: torch.dtype = F32) -> torch.Tensor:
    return torch.empty(shape, dtype=F32, device=DEVICE).normal_(mean, std, generator=g).to(dtype)


def _fp8(g: torch.Generator, rows: int, width: int) -> torch.Tensor:
    """Normal values in e4m3, the largest of a block near the type's largest; rows start on 16 bytes."""
    store = torch.zeros((rows, -(-width // 16) * 16), dtype=E4M3, device=DEVICE)
    store[:, :width] = _normal(g, rows, width, std=150.0).clamp_(-TOP, TOP).to(E4M3)
    return store[:, :width]


def prepare(case: dict, seed: int) -> dict:
    g = _generator(seed)
    kind, rows, dtype = case["kind"], case["rows"], TYPES[case["type"]]
    if kind == "logprobs":
        v = case["vocabulary"]
        logits = _normal(g, rows, v, std=2.5)
        likely = torch.randint(0, v, (rows, 8), generator=g, device=DEVICE)  # a few tokens stand out in every row
        logits.scatter_add_(1, likely, _normal(g, rows, 8, std=4.0, mean=10.0))
        # half of the tokens in question are likely ones, the others are any
        tokens = torch.where(torch.rand(rows, generator=g, device=DEVICE) < 0.5, likely[:, 0], torch.randint(0, v, (rows,), generator=g, device=DEVICE))
        if case["masked"]:
            keep = torch.rand((rows, v), generator=g, device=DEVICE) >= case["masked"]
            keep.scatter_(1, tokens[:, None], True)
            logits.masked_fill_(~keep, -math.inf)
        return dict(kind=kind, logits=logits.to(dtype), tokens=tokens, top=case["top"])
    width = case["width"]
    if kind == "quantize":
        x = _normal(g, rows, case["stride"], dtype=dtype)
        x *= _normal(g, rows, 1, std=0.5).exp().to(dtype)  # tokens (or features) differ in size
        if rows > 4:
            x[rows // 2] = 0  # a row of padding
        return dict(kind=kind, form=case["form"], x=x[:, :width])
    if kind == "norm":
        residual = _normal(g, rows, width, std=3.0)
        residual[:, :: max(1, width // 7)] *= 6.0  # a few features of a stream are large in every token
        return dict(kind=kind, residual=residual, delta=_normal(g, rows, width, dtype=dtype), out=torch.empty_like(residual),
                    weight=_normal(g, width, std=0.1, mean=1.0, dtype=TYPES[case["weight"]]))
    features, k_blocks = case["features"], _blocks(width)
    stacked = 2 * BLOCK * _blocks(features) if kind == "gated" else features
    x, w = _fp8(g, rows, width), _fp8(g, stacked, width)
    x_scales = (0.007 * _normal(g, k_blocks, rows, std=0.3).exp()).t()  # (the tokens of a block of columns stand side by side)
    w_scales = 0.007 / math.sqrt(width) * _normal(g, _blocks(stacked), k_blocks, std=0.3).exp()
    bias = _normal(g, stacked, dtype=BF16) if case["bias"] else None
    return dict(kind=kind, x=x, x_scales=x_scales, w=w, w_scales=w_scales, bias=bias, type=dtype, features=features)


# --------------------------------------------------------------------------- the operators

def _plain_scales(top: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(what values are multiplied by, the scale) of blocks whose largest magnitude is ``top``."""
    largest = torch.full_like(top, TOP)
    return torch.where(top > 0, largest / top, torch.zeros_like(top)), top / largest


def _plain_fp8(v: torch.Tensor, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """float32 [N, K] to the e4m3 values (kept in float32) and the scales of blocks of ``rows`` x 128."""
    n, k = v.shape
    padded = v.new_zeros((-(-n // rows) * rows, _blocks(k) * BLOCK))
    padded[:n, :k] = v
    tiles = padded.reshape(-1, rows, _blocks(k), BLOCK)
    inverse, scales = _plain_scales(tiles.abs().amax(dim=(1, 3), keepdim=True))
    q = (tiles * inverse).to(E4M3).float().reshape(padded.shape)[:n, :k]
    return q, scales[:, 0, :, 0]


def _plain_values(q: torch.Tensor, scales: torch.Tensor, rows: int) -> torch.Tensor:
    full = scales.repeat_interleave(BLOCK, dim=1)[:, : q.shape[1]]
    return q.float() * (full if rows == 1 else full.repeat_interleave(rows, dim=0)[: q.shape[0]])


def _plain_logprobs(state: dict):
    z, tokens, k = state["logits"].float(), state["tokens"], state["top"]
    v = z.shape[1]
    shifted = z - z.amax(dim=1, keepdim=True)
    p = shifted.exp()
    total = p.sum(dim=1, keepdim=True, dtype=F64)
    log_total = total.log()
    entropy = log_total - torch.where(p > 0, p * shifted, torch.zeros_like(p)).sum(dim=1, keepdim=True, dtype=F64) / total
    own_z = z.gather(1, tokens[:, None])
    logprob = shifted.gather(1, tokens[:, None]) - log_total
    index = torch.arange(v, device=z.device)
    ahead = (z > own_z) | ((z == own_z) & (index < tokens[:, None]))
    out = [logprob[:, 0].float(), entropy[:, 0].float(), (1 + ahead.sum(dim=1)).int()]
    if k:
        # whole numbers in the order of the values (+ 0.0: both zeros are one), the lower index first among equals
        bits = (z + 0.0).view(torch.int32).long()
        order = torch.where(bits >= 0, bits, -2147483648 - bits) * (1 << 32) - index
        at = order.topk(k, dim=1).indices
        out += [(shifted.gather(1, at) - log_total).float(), at.int()]
    return tuple(out)


def _plain(state: dict):
    kind = state["kind"]
    if kind == "logprobs":
        return _plain_logprobs(state)
    if kind == "quantize":
        rows = 1 if state["form"] == "rows" else BLOCK
        q, scales = _plain_fp8(state["x"].float(), rows)
        return _plain_values(q, scales, rows).to(BF16), scales
    if kind == "norm":
        stream = state["residual"] + state["delta"].float()
        normed = stream * torch.rsqrt((stream * stream).mean(dim=1, keepdim=True) + EPS) * state["weight"].float()
        q, scales = _plain_fp8(normed, 1)
        return stream, _plain_values(q, scales, 1).to(BF16), scales
    y = _plain_values(state["x"], state["x_scales"], 1) @ _plain_values(state["w"], state["w_scales"], BLOCK).t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    if kind == "gated":
        runs = y.reshape(y.shape[0], -1, 2, BLOCK)
        gate, up = runs[:, :, 0].reshape(y.shape[0], -1), runs[:, :, 1].reshape(y.shape[0], -1)
        y = (gate / (1.0 + torch.exp(-gate)) * up)[:, : state["features"]]
        if state["type"] == E4M3:
            q, scales = _plain_fp8(y, 1)
            return _plain_values(q, scales, 1).to(BF16), scales
    return y.to(state["type"])


def _kernels(state: dict):
    from slipstream_b200 import ops

    kind = state["kind"]
    if kind == "logprobs":
        r = ops.token_logprobs(state["logits"], state["tokens"], top=state["top"])
        return (r.logprobs, r.entropy, r.ranks, *((r.top_logprobs, r.top_tokens) if state["top"] else ()))
    if kind == "quantize":
        q = ops.quantize_rows_fp8(state["x"]) if state["form"] == "rows" else ops.quantize_blocks_fp8(state["x"])
        return ops.dequantize_fp8(q, BF16), q.scales
    if kind == "norm":
        q = ops.add_rmsnorm_fp8(state["residual"], state["delta"], state["weight"], EPS, residual_out=state["out"])
        return state["out"], ops.dequantize_fp8(q, BF16), q.scales
    x, w = ops.Fp8Rows(state["x"], state["x_scales"]), ops.Fp8Blocks(state["w"], state["w_scales"])
    if kind == "linear":
        return ops.linear_fp8(x, w, state["bias"], state["type"])
    y = ops.gate_up_swiglu_fp8(x, w, state["bias"], state["type"], features=state["features"])
    return (ops.dequantize_fp8(y, BF16), y.scales) if state["type"] == E4M3 else y


def run(state: dict):
    return _kernels(state) if own else _plain(state)


# --------------------------------------------------------------------------- what a pass needs, and what is exact

def work(case: dict) -> dict:
    rows, size = case["rows"], SIZES[case["type"]]
    if case["kind"] == "logprobs":
        n = rows * case["vocabulary"]
        return {"bytes": n * size + rows * (8 + 12 + 8 * case["top"]), "flops": 7 * n}
    width = case["width"]
    if case["kind"] == "quantize":  # the rows in; e4m3, the scales and the values they stand for out
        scales = (rows if case["form"] == "rows" else _blocks(rows)) * _blocks(width)
        return {"bytes": rows * width * (size + 1 + 2) + 4 * scales, "flops": 3 * rows * width}
    if case["kind"] == "norm":  # stream and branch in; stream, e4m3, scales and values out
        return {"bytes": rows * (width * (4 + size + 4 + 1 + 2) + 4 * _blocks(width)) + width * SIZES[case["weight"]], "flops": 8 * rows * width}
    features = case["features"]
    stacked = 2 * features if case["kind"] == "gated" else features
    out = rows * features * size
    if case["type"] == "fp8":  # e4m3, scales and the values they stand for
        out += rows * (2 * features + 4 * _blocks(features))
    scales = 4 * _blocks(width) * (rows + _blocks(stacked))
    return {"bytes": rows * width + stacked * width + scales + (2 * stacked if case["bias"] else 0) + out, "flops": 2 * rows * stacked * width}


def _to_e4m3(v: torch.Tensor) -> torch.Tensor:
    """float64 to the nearest e4m3, ties to even: eight steps in each power of two, none finer than 2^-9."""
    exponent = torch.frexp(v.abs())[1] - 1
    step = torch.ldexp(torch.ones_like(v), torch.clamp(exponent, min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _exact_fp8(v: torch.Tensor, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Values that float64 [N, K] in e4m3 stands for, and the scales; a block of columns after the other."""
    out, scales = torch.zeros_like(v), torch.zeros((-(-v.shape[0] // rows), _blocks(v.shape[1])), dtype=F64, device=v.device)
    owner = torch.arange(v.shape[0], device=v.device) // rows
    for b in range(scales.shape[1]):
        part = v[:, b * BLOCK: (b + 1) * BLOCK]
        top = torch.zeros_like(scales[:, 0]).scatter_reduce(0, owner, part.abs().max(dim=1).values, "amax")
        scales[:, b] = top / TOP
        scale = scales[:, b][owner][:, None]
        out[:, b * BLOCK: (b + 1) * BLOCK] = torch.where(scale > 0, _to_e4m3(part / scale.clamp(min=1e-300)) * scale, torch.zeros_like(part))
    return out, scales


def _exact_logprobs(state: dict, k: int):
    rows = []
    for z, token in zip(state["logits"], state["tokens"].tolist()):
        z = z.to(F64)
        log_p = torch.log_softmax(z, dim=0)
        kept = log_p[z > -math.inf]
        before = int((z[:token] >= z[token]).sum()) + int((z[token + 1:] > z[token]).sum())
        order = torch.sort(z, descending=True, stable=True).indices[:k]
        rows.append((log_p[token], -(kept.exp() * kept).sum(), before + 1, log_p[order], order))
    columns = list(zip(*rows))
    out = [torch.stack(columns[0]), torch.stack(columns[1]), torch.tensor(columns[2], dtype=torch.int32, device=DEVICE)]
    return tuple(out + [torch.stack(columns[3]), torch.stack(columns[4]).int()] if k else out)


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "logprobs":
        return _exact_logprobs(state, case["top"])
    if kind == "quantize":
        return _exact_fp8(state["x"].to(F64), 1 if case["form"] == "rows" else BLOCK)
    if kind == "norm":
        stream = state["residual"].to(F64) + state["delta"].to(F64)
        v = stream / (stream.square().sum(dim=1, keepdim=True) / case["width"] + EPS).sqrt() * state["weight"].to(F64)
        return (stream, *_exact_fp8(v, 1))
    features, out = torch.arange(state["w"].shape[0], device=DEVICE), None
    for b in range(_blocks(case["width"])):
        cut = slice(b * BLOCK, (b + 1) * BLOCK)
        part = torch.matmul(state["x"][:, cut].to(F64), state["w"][:, cut].to(F64).mT)
        part *= torch.outer(state["x_scales"][:, b].to(F64), state["w_scales"][:, b].to(F64)[features // BLOCK])
        out = part if out is None else out + part
    if state["bias"] is not None:
        out = out + state["bias"].to(F64)
    if kind == "linear":
        return out
    at = torch.arange(case["features"], device=DEVICE)
    at = at // BLOCK * (2 * BLOCK) + at % BLOCK
    gate, up = out[:, at], out[:, at + BLOCK]
    out = gate * torch.sigmoid(gate) * up
    return _exact_fp8(out, 1) if case["type"] == "fp8" else out
