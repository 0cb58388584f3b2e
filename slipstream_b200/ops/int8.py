"""Rows of 8-bit integers: the norm that ends in them, products of them, and how values become them and back.

A row of int8 values comes with one float32 scale and stands for ``values * scale``.  Activations are such rows (a scale per
token), and so are the weights of a product (a scale per output feature).  A product of both is exact in 32-bit integers; the
scales are applied to the sum.  ``quantize_rows_int8`` is symmetric and has no zero point: the largest magnitude of a row becomes
127 (or -127), a row of zeros has the scale 0, and a row that holds an infinity or NaN has the scale NaN, so that what is formed
from it is NaN.

Rows of values start on 16 bytes: their stride is a multiple of 16, whatever their width.  The functions here that return int8 rows make
them so (csrc/int8_calls.cpp), in one allocation, the scales behind the values: what keeps or saves either keeps or saves both.
`int8_rows_like` makes rows in two allocations, for a program that fills them itself.

Weights, their scales, biases and the weights of a norm are taken for constant, as elsewhere in this package: a kernel may read them
before the kernels in front of it are through.  `quantize_rows_int8` and `dequantize_rows_int8` therefore keep the kernels behind them
waiting unless they are told (``activations=True``) that what they write will not be a product's weights.  The results of the norm and
of products are activations.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from .functions import KernelError, _native_launches, error_word, gemm_library, ops_library, sm_count
from .library import load_calls

RUN = 64  # gate and up rows of a stacked weight alternate in runs of this many (csrc/int8_calls.cpp)
_BF16 = torch.bfloat16


class Int8Rows:
    """``values`` int8 [N, K], whose rows start on 16 bytes, and ``scales`` float32 [N]: row n stands for
    ``values[n] * scales[n]``."""

    __slots__ = ("values", "scales")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor) -> None:
        self.values = values
        self.scales = scales

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def device(self) -> torch.device:
        return self.values.device

    def nbytes(self) -> int:
        """Bytes a pass over the rows reads (without what pads them)."""
        return self.values.numel() + 4 * self.scales.numel()

    def dequantize(self, dtype: torch.dtype, *, activations: bool = False) -> torch.Tensor:
        return dequantize_rows_int8(self, dtype, activations=activations)


_native = None


def _calls():
    """The calls' host side (csrc/int8_calls.cpp), loaded and told its entry points at the first call."""
    global _native
    if _native is None:
        ops, gemm, module = ops_library(), gemm_library(), load_calls()
        entries = [ctypes.cast(f, ctypes.c_void_p).value for f in (ops.ss_quantize_rows_int8, ops.ss_dequantize_rows_int8,
                                                                   ops.ss_add_rmsnorm_int8, gemm.ss_gemm_int8)]
        module.use(KernelError, *entries, _error_address, _plan_on)
        if module.launched not in _native_launches:  # (two threads may make the first call)
            _native_launches.append(module.launched)
        _native = module
    return _native


def _error_address(index: int) -> int:
    return error_word(torch.device("cuda", index)).data_ptr()  # (the word lives as long as the process)


@functools.lru_cache(maxsize=None)
def _resident(index: int) -> tuple[tuple[int, ...], tuple[int, ...]]:
    """How many clusters of 1 to 8 blocks of the product of few tokens the device holds at the same time, with its ring sized for
    one block an SM and for two."""
    lib, sms = gemm_library(), sm_count(index)
    with torch.cuda.device(index):
        return tuple(tuple(lib.ss_gemm_int8_resident(n, per) or sms * per // n for n in range(1, 9)) for per in (1, 2))


def _plan_on(tokens: int, features: int, k: int, gated: int, index: int) -> tuple[int, int, int, int, int]:
    return int8_plan(tokens, features, k, sm_count(index), bool(gated), _resident(index))


def int8_rows_like(rows: int, width: int, device: torch.device) -> Int8Rows:
    """Int8 rows with nothing in them yet, for a program that fills them itself."""
    values = torch.empty_strided((rows, width), ((width + 15) & -16, 1), dtype=torch.int8, device=device)
    return Int8Rows(values, torch.empty(rows, dtype=torch.float32, device=device))


def _need_rows(r: Int8Rows, what: str) -> None:
    if not isinstance(r, Int8Rows):
        raise KernelError(f"{what} must be Int8Rows, not {type(r).__name__}")


def quantize_rows_int8(x: torch.Tensor, *, activations: bool = False) -> Int8Rows:
    """The rows of ``x`` (float32 or bfloat16 [N, K], any row stride) as int8 rows: ``a = max |x_n|``, ``scale = a / 127``,
    ``q = rint(x * (127 / a))`` in float32, ties to even.  Tokens of activations, or output features of a weight.

    ``activations``: the rows are a product's activations, not its weights, and the kernel behind may start early."""
    return Int8Rows(*(_native or _calls()).quantize(x, activations))


def dequantize_rows_int8(rows: Int8Rows, dtype: torch.dtype, *, activations: bool = False) -> torch.Tensor:
    """``values * scales`` as a tensor [N, K] of ``dtype`` (float32 or bfloat16), rounded once.

    ``activations``: the tensor is a product's activations, not its weights, and the kernel behind may start early."""
    _need_rows(rows, "rows")
    return (_native or _calls()).dequantize(rows.values, rows.scales, dtype, activations)


def add_rmsnorm_int8(residual: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor, eps: float, *,
                     residual_out: torch.Tensor | None = None) -> Int8Rows:
    """``add_rmsnorm`` that ends in int8 rows: ``residual`` (float32 [N, H]) += ``delta`` (float32 or bfloat16, or None), and
    ``x / sqrt(mean(x^2) + eps) * weight`` of the new stream, formed in float32 (from ``x * weight``, which has to be finite), as int8 rows.

    ``residual_out`` (float32 [N, H]) gets the new stream instead, and ``residual`` stays as it is.  ``weight`` is bfloat16 or
    float32.  A row's result does not depend on the other rows, nor on how many there are."""
    return Int8Rows(*(_native or _calls()).norm(residual, delta, weight, eps, residual_out))


# --------------------------------------------------------------------------- products

def int8_plan(tokens: int, features: int, k: int, sms: int, gated: bool = False,
              resident: tuple[tuple[int, ...], tuple[int, ...]] | None = None) -> tuple[int, int, int, int, int]:
    """(many, tile, K slices, blocks an SM, steps) of ``x[tokens, k] @ w[features, k].T``: which of the two kernels, the width of its
    tile (tokens of the first, features of the second), for the first the slices of K and how many blocks an SM the ring is sized
    for, and for both how many steps of K a stage holds.  ``resident``: clusters of 1 to 8 blocks that run at the same time, with the
    ring sized for one block an SM and for two.

    The choice is the cheapest by an estimate of cycles whose constants are fitted to 9,592 measured products (1 to 4,096 tokens, the
    projections of the 0.5B, 1.5B and 7B layer sizes, tiles, slices and stages of all sizes).  What it takes is on average 2 % slower
    than the fastest of them at the same sizes, and at worst 17 %; one tile for all tokens up to 256 with K in one slice, else tiles of
    256 x 256, would be 42 % slower."""
    # what follows depends on the tokens in steps of 16 (their tiles) up to 640 and of 256 beyond: few plans for many counts
    step = 16 if tokens <= 640 else 256
    return _plan((tokens + step - 1) // step * step, features, k, sms, gated, resident)


@functools.lru_cache(maxsize=None)
def _plan(tokens: int, features: int, k: int, sms: int, gated: bool, resident) -> tuple[int, int, int, int, int]:
    if resident is None:
        resident = tuple(tuple(sms * per // n for n in range(1, 9)) for per in (1, 2))
    k_steps = (k + 127) // 128
    best = None
    few = tokens <= 640 and (features + 127) // 128 <= 65535  # (its tiles of features are blocks along grid.y)
    for parts in range(1, 9) if few else ():
        tile = ((tokens + parts - 1) // parts + 15) // 16 * 16
        if tile > 256 or (parts > 1 and tile <= 16):
            continue
        tiles = (features + 127) // 128 * ((tokens + tile - 1) // tile)
        for slices in range(1, min(8, k_steps) + 1):
            blocks = tiles * slices
            if slices > 1 and blocks > 3 * sms:
                break
            if slices == 7:  # (clusters that fit worst into the GPU's processor clusters)
                continue
            for per, steps in ((1, 1), (1, 2), (2, 1), (2, 2)) if tile <= 128 else ((1, 1), (1, 2)):
                rest = 2560 + ((tile + slices - 1) // slices * 512 if slices > 1 else 0)
                stages = min(12, ((232448 if per == 1 else 115712) - rest) // (steps * (128 + tile) * 128))
                if stages < 2:
                    continue
                held = max(1, resident[per - 1][slices - 1]) * slices  # blocks that run at the same time
                waves = (blocks + held - 1) // held
                shared = max(1.0, min(float(per), blocks / sms))
                # a step of K: the loops of the fetching and issuing threads; what an SM takes in; the ring's latency; the memory
                cycles = max(537.0 if steps == 1 else 235.0, shared * (128 + tile) * 128 / 60, 2905 / (stages * steps),
                             min(blocks, held) * 16384 * 148 / (5155 * sms))
                mine = (k_steps + slices * steps - 1) // (slices * steps) * steps
                cost = 3190 + waves * (mine * cycles + 12 + 41.5 * tile)
                if slices > 1:
                    cost += waves * 107.6 * tile * (slices - 1) / slices
                if waves > 1:
                    cost += 540
                elif per == 2 and blocks <= (0.5 if slices == 1 else 0.45) * held:  # the kernel behind has room for its first stages
                    cost -= 2970
                if best is None or cost < best[0]:
                    best = (cost, (0, tile, slices, per, steps))
    if tokens > 64 or not few:
        rows = (tokens + 255) // 256
        for tile in ((128, 256) if gated else (32, 64, 96, 128, 160, 192, 224, 256)):
            tiles = rows * ((features + tile - 1) // tile)
            pairs = max(1, sms // 2)
            rounds = (tiles + pairs - 1) // pairs
            for steps in (1, 2):
                cycles = max(411.0 if steps == 1 else 230.0, (2.06 if steps == 1 else 2.78) * tile,
                             min(tiles, pairs) * tile * 128 * 148 / (5155 * sms * min(rows, pairs)))
                cost = 10450 + rounds * k_steps * cycles + 6.8 * tile + (rounds - 1) * 750
                if best is None or cost < best[0]:
                    best = (cost, (1, tile, 1, 1, steps))
    return best[1]


def linear_int8(x: Int8Rows, weight: Int8Rows, bias: torch.Tensor | None = None, out_dtype: torch.dtype = _BF16, *,
                plan: tuple[int, int, int, int, int] | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` for int8 rows: ``x`` [tokens, K] with a scale a token, ``weight`` [features, K] with a scale a
    feature.  The sum over K (up to 131,071 elements) is exact, in 32-bit integers; it is multiplied by both scales and the bias
    (bfloat16 or float32 [features]) is added in float32, and the result is rounded once to ``out_dtype`` (bfloat16 or float32).
    ``plan``: see `int8_plan`; every plan gives the same bits."""
    _need_rows(x, "x")
    _need_rows(weight, "weight")
    return (_native or _calls()).product(x.values, x.scales, weight.values, weight.scales, bias, out_dtype, False, None, plan)


def gate_up_swiglu_int8(x: Int8Rows, weight: Int8Rows, bias: torch.Tensor | None = None, out_dtype: torch.dtype = _BF16, *,
                        features: int | None = None, plan: tuple[int, int, int, int, int] | None = None) -> torch.Tensor:
    """``silu(gate(x)) * up(x)`` for int8 rows, the products as in `linear_int8`, the unit formed in float32 in the product's
    epilogue and rounded once.  The rows of ``weight`` (and of ``bias``) alternate ``RUN`` gate and ``RUN`` up features
    (`stack_gate_up`); ``features``: how many of the weight's pairs are real (those behind them pad the last run)."""
    _need_rows(x, "x")
    _need_rows(weight, "weight")
    return (_native or _calls()).product(x.values, x.scales, weight.values, weight.scales, bias, out_dtype, True, features, plan)


def stack_gate_up(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """The rows of ``gate`` and ``up`` (matrices or vectors of I rows) in alternating runs of ``RUN``, the last run padded with
    zeros: the layout of `gate_up_swiglu_int8`, for weights before they are rounded and for biases."""
    if gate.shape != up.shape:
        raise KernelError(f"gate {tuple(gate.shape)} and up {tuple(up.shape)} differ")
    rows, rest = gate.shape[0], gate.shape[1:]
    runs = -(-rows // RUN)
    stacked = gate.new_zeros((runs, 2, RUN, *rest))
    for i, t in enumerate((gate, up)):
        padded = t.new_zeros((runs * RUN, *rest))
        padded[:rows] = t
        stacked[:, i] = padded.reshape(runs, RUN, *rest)
    return stacked.reshape(2 * runs * RUN, *rest)


__all__ = ["Int8Rows", "int8_rows_like", "quantize_rows_int8", "dequantize_rows_int8", "add_rmsnorm_int8", "linear_int8",
           "gate_up_swiglu_int8", "stack_gate_up", "int8_plan"]
