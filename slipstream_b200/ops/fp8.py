"""Rows and weights in 8-bit floats (e4m3) with a float32 scale for each block of 128: the norm that ends in them, products of them, and how
values become them and back.

Activations are `Fp8Rows`: a scale for each row and each 128 of its elements.  Weights are `Fp8Blocks`: a scale for each 128 rows x
128 columns.  A block of values v becomes ``scale = a / 448``, ``a = max |v|``, and ``q = e4m3(v * (448 / a))``, ties to even; it stands
for ``q * scale``.  A block of zeros has the scale 0; a block that holds an infinity or NaN has the scale NaN (and q = 0), so that what
is formed from it is NaN.

Rows of values start on 16 bytes: their stride is a multiple of 16, whatever their width.  The functions here that return such rows or
blocks make them so (csrc/fp8_calls.cpp), in one allocation, the scales behind the values: what keeps or saves either keeps or saves
both.  Scales may have any strides.

Weights, their scales, biases and the weights of a norm are taken for constant, as elsewhere in this package: a kernel may read them
before the kernels in front of it are through.  `quantize_rows_fp8` and `dequantize_fp8` therefore keep the kernels behind them waiting
unless they are told (``activations=True``) that what they write will not be a product's weights; `quantize_blocks_fp8` always does.
The results of the norm and of products are activations.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from .functions import KernelError, _native_launches, error_address, fp8_library, sm_count
from .library import load_calls

FP8_BLOCK = 128  # elements that share a scale; gate and up rows of a stacked weight alternate in runs of as many (csrc/fp8_calls.h)
_BF16 = torch.bfloat16


class _Scaled:
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
        """Bytes a pass over the values and scales reads (without what pads them)."""
        return self.values.numel() + 4 * self.scales.numel()

    def dequantize(self, dtype: torch.dtype, *, activations: bool = False) -> torch.Tensor:
        return dequantize_fp8(self, dtype, activations=activations)


class Fp8Rows(_Scaled):
    """``values`` float8_e4m3fn [N, K], whose rows start on 16 bytes, and ``scales`` float32 [N, ceil(K / 128)]: element (n, k) stands
    for ``values[n, k] * scales[n, k // 128]``."""

    __slots__ = ()


class Fp8Blocks(_Scaled):
    """``values`` float8_e4m3fn [F, K], whose rows start on 16 bytes, and ``scales`` float32 [ceil(F / 128), ceil(K / 128)]: element
    (f, k) stands for ``values[f, k] * scales[f // 128, k // 128]``."""

    __slots__ = ()


_native = None


def _calls():
    """The calls' host side (csrc/fp8_calls.cpp), loaded and told its entry points at the first call."""
    global _native
    if _native is None:
        lib, module = fp8_library(), load_calls("fp8_calls")
        entries = [ctypes.cast(f, ctypes.c_void_p).value for f in (lib.ss_quantize_fp8, lib.ss_dequantize_fp8, lib.ss_add_rmsnorm_fp8, lib.ss_gemm_fp8)]
        module.use(KernelError, *entries, error_address, _plan_on)
        if module.launched not in _native_launches:  # (two threads may make the first call)
            _native_launches.append(module.launched)
        _native = module
    return _native


@functools.lru_cache(maxsize=None)
def _resident(index: int) -> tuple[tuple[int, ...], tuple[int, ...]]:
    """How many clusters of 1 to 8 blocks of the product of few tokens the device holds at the same time, with its ring sized for
    one block an SM and for two."""
    lib, sms = fp8_library(), sm_count(index)
    with torch.cuda.device(index):
        return tuple(tuple(lib.ss_gemm_fp8_resident(n, per) or sms * per // n for n in range(1, 9)) for per in (1, 2))


def _plan_on(tokens: int, features: int, k: int, gated: int, index: int) -> tuple[int, int, int, int]:
    return fp8_plan(tokens, features, k, sm_count(index), bool(gated), _resident(index))


def _need(r: _Scaled, kind: type, what: str) -> None:
    if not isinstance(r, kind):
        raise KernelError(f"{what} must be {kind.__name__}, not {type(r).__name__}")


def quantize_rows_fp8(x: torch.Tensor, *, activations: bool = False) -> Fp8Rows:
    """The rows of ``x`` (float32 or bfloat16 [N, K], any row stride) as fp8 rows, formed in float32.

    ``activations``: the rows are a product's activations (nothing else reads them early), and the kernel behind may start early."""
    return Fp8Rows(*(_native or _calls()).quantize(x, False, activations))


def quantize_blocks_fp8(x: torch.Tensor) -> Fp8Blocks:
    """``x`` (float32 or bfloat16 [F, K], any row stride) with a scale for each 128 x 128 elements: a product's weight."""
    return Fp8Blocks(*(_native or _calls()).quantize(x, True, False))


def dequantize_fp8(x: Fp8Rows | Fp8Blocks, dtype: torch.dtype, *, activations: bool = False) -> torch.Tensor:
    """``values * scales`` as a tensor of ``dtype`` (float32 or bfloat16), rounded once.

    ``activations``: the tensor is a product's activations, not its weights, and the kernel behind may start early."""
    _need(x, _Scaled, "x")
    return (_native or _calls()).dequantize(x.values, x.scales, isinstance(x, Fp8Blocks), dtype, activations)


def add_rmsnorm_fp8(residual: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor, eps: float, *,
                    residual_out: torch.Tensor | None = None) -> Fp8Rows:
    """``add_rmsnorm`` that ends in fp8 rows: ``residual`` (float32 [N, H]) += ``delta`` (float32 or bfloat16, or None), and
    ``x / sqrt(mean(x^2) + eps) * weight`` of the new stream, formed in float32 (from ``x * weight``, which has to be finite), as fp8 rows.

    ``residual_out`` (float32 [N, H]) gets the new stream instead, and ``residual`` stays as it is.  ``weight`` is bfloat16 or
    float32.  A row's result does not depend on the other rows, nor on how many there are."""
    return Fp8Rows(*(_native or _calls()).norm(residual, delta, weight, eps, residual_out))


# --------------------------------------------------------------------------- products

def fp8_plan(tokens: int, features: int, k: int, sms: int, gated: bool = False,
             resident: tuple[tuple[int, ...], tuple[int, ...]] | None = None) -> tuple[int, int, int, int]:
    """(many, tile, K slices, blocks an SM) of ``x[tokens, k] @ w[features, k].T``: which of the two kernels, the width of its tile
    (tokens of the first, features of the second), the slices of K, and for the first how many blocks an SM the ring is sized for.
    ``resident``: clusters of 1 to 8 blocks that run at the same time, with the ring sized for one block an SM and for two.

    The choice is the cheapest by an estimate in microseconds whose constants are fitted to 2,772 measured products (1 to 512 tokens, the
    projections of the 0.5B, 1.5B and 7B layer sizes, tiles, slices and rings of all sizes): on average 2 % slower than the fastest of
    them at the same sizes, and at worst 16 % (48 tokens of 1,536 x 8,960 gated); those of the second kernel with K in slices to 564 more (256 x 18,944 x 3,584: 54 us in
    one slice, 31 in five)."""
    # what follows depends on the tokens in steps of 16 (their tiles) up to 640 and of 256 beyond: few plans for many counts
    step = 16 if tokens <= 640 else 256
    return _plan((tokens + step - 1) // step * step, features, k, sms, gated, resident)


def _few_rest(tile: int, slices: int, gated: bool) -> int:
    """Bytes of shared memory that a block of the kernel for few tokens has beside its ring (csrc/gemm_fp8.cu, launch_few)."""
    parts = 2 if gated else 1
    half = next(c for c in (8, 16, 32, 64, 128) if 2 * c >= tile)
    floats = (8 if parts * half <= 32 else 4) * ((half + parts + 3) // 4 * 4) + 2 * parts * half
    return 1536 + 32 * floats + (slices * ((tile + slices - 1) // slices) * 512 * parts if slices > 1 else 0)


@functools.lru_cache(maxsize=None)
def _plan(tokens: int, features: int, k: int, sms: int, gated: bool, resident) -> tuple[int, int, int, int]:
    if resident is None:
        resident = tuple(tuple(sms * per // n for n in range(1, 9)) for per in (1, 2))
    blocks = (k + 127) // 128
    parts = 2 if gated else 1  # 128 rows of the weight in a tile of the kernel for few tokens
    best = None
    down = (features + 128 * parts - 1) // (128 * parts)
    few = tokens <= 640 and (features + 127) // 128 <= 65535  # (its tiles of features are blocks along grid.y)
    for tile in (16, 32, 48, 64, 96, 128) if few else ():
        across = (tokens + tile - 1) // tile
        if tile > 128 // parts or across > 8 or (tile > 16 and tile >= tokens + 16):
            continue
        for slices in range(1, min(8, blocks) + 1):
            count = down * across * slices
            if slices > 1 and count > 3 * sms:
                break
            if slices == 7:  # (clusters that fit worst into the GPU's processor clusters)
                continue
            alone = max(1, resident[0][slices - 1]) * slices  # blocks that run at the same time, one an SM
            # (two blocks an SM: only so that the kernel behind has room for its first copies, never for more blocks of this one)
            for per in (1, 2) if tile <= 64 and not gated and count <= alone else (1,):
                stage = (128 * parts + tile) * 128
                stages = min(12, ((232448 if per == 1 else 115712) - _few_rest(tile, slices, gated)) // stage)
                if stages < (2 if slices > 1 else -(-tile * 512 * parts // stage)):
                    continue
                waves = (count + alone - 1) // alone
                # a block of K: the loops of the threads and the sums that they take out; the ring's latency; the memory
                each = max(0.244 + 0.0033 * tile * parts, 1.09 / stages, min(count, alone) * 16384 * parts * 0.136e-6 * 148 / sms)
                cost = 0.243 + waves * ((blocks + slices - 1) // slices * each + 1.81 + 0.0443 * tile * parts)
                if slices > 1:
                    cost += waves * (1.75 + 0.0087 * tile * parts * (slices - 1) / slices)
                if waves > 1:
                    cost += 0.175
                elif per == 2:
                    cost -= 0.267
                if best is None or cost < best[0]:
                    best = (cost, (0, tile, slices, per))
    if tokens > 32 or not few:
        rows = (tokens + 255) // 256
        for tile in ((256,) if gated else (64, 128, 256)):
            tiles = rows * ((features + tile - 1) // tile)
            pairs = max(1, sms // 2)
            for slices in (1,) if gated or tile == 64 else range(1, max(1, min(8, blocks // 2)) + 1):
                if slices > 1 and tiles * slices > 2 * pairs:
                    break
                rounds = (tiles * slices + pairs - 1) // pairs
                cost = 3.89 + rounds * ((blocks + slices - 1) // slices * (0.204 + 0.000926 * tile) + 0.138 + 0.0123 * tile)
                if slices > 1:  # another launch, the parts written and read again
                    cost += 3.19 + (0.226 * slices + 0.507) * tokens * features * 4e-6
                if best is None or cost < best[0]:
                    best = (cost, (1, tile, slices, 1))
    return best[1]


def linear_fp8(x: Fp8Rows, weight: Fp8Blocks, bias: torch.Tensor | None = None, out_dtype: torch.dtype = _BF16, *,
               plan: tuple[int, int, int, int] | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` for fp8 operands: ``x`` [tokens, K], ``weight`` [features, K].  The sum over each block of 128 of K is
    formed by the tensor cores in float32, multiplied by the product of both scales and added up in float32; the bias (bfloat16 or
    float32 [features]) is added last, and the result is rounded once to ``out_dtype`` (bfloat16 or float32).
    ``plan``: see `fp8_plan`; plans that cut K into other slices add the blocks' sums in another order."""
    _need(x, Fp8Rows, "x")
    _need(weight, Fp8Blocks, "weight")
    if out_dtype == torch.float8_e4m3fn:
        raise KernelError("linear_fp8 writes float32 or bfloat16")
    return (_native or _calls()).product(x.values, x.scales, weight.values, weight.scales, bias, out_dtype, False, None, plan)


def gate_up_swiglu_fp8(x: Fp8Rows, weight: Fp8Blocks, bias: torch.Tensor | None = None, out_dtype: torch.dtype = _BF16, *,
                       features: int | None = None, plan: tuple[int, int, int, int] | None = None) -> torch.Tensor | Fp8Rows:
    """``silu(gate(x)) * up(x)`` for fp8 operands, the products as in `linear_fp8`, the unit formed in float32 in the product's epilogue
    and rounded once: to bfloat16 or float32, or (``out_dtype`` float8_e4m3fn) to fp8 rows, as `quantize_rows_fp8` does.  (But for float32
    outputs the exponential and the division are the approximate ones, off by about 2^-21.)
    The rows of ``weight`` (and of ``bias``) alternate ``FP8_BLOCK`` gate and ``FP8_BLOCK`` up features (`stack_gate_up_fp8`);
    ``features``: how many of the weight's pairs are real (those behind them pad the last run)."""
    _need(x, Fp8Rows, "x")
    _need(weight, Fp8Blocks, "weight")
    out = (_native or _calls()).product(x.values, x.scales, weight.values, weight.scales, bias, out_dtype, True, features, plan)
    return Fp8Rows(*out) if type(out) is tuple else out


def stack_gate_up_fp8(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """The rows of ``gate`` and ``up`` (matrices or vectors of I rows) in alternating runs of ``FP8_BLOCK``, the last run padded with
    zeros: the layout of `gate_up_swiglu_fp8`, for weights before they are rounded and for biases.  A run is a block of the scales'
    own, so the scales of matrices that were rounded before, stacked alike, stay theirs."""
    if gate.shape != up.shape:
        raise KernelError(f"gate {tuple(gate.shape)} and up {tuple(up.shape)} differ")
    rows, rest = gate.shape[0], gate.shape[1:]
    runs = -(-rows // FP8_BLOCK)
    stacked = gate.new_zeros((runs, 2, FP8_BLOCK, *rest))
    for i, t in enumerate((gate, up)):
        whole = rows // FP8_BLOCK
        stacked[:whole, i] = t[: whole * FP8_BLOCK].reshape(whole, FP8_BLOCK, *rest)
        if whole < runs:
            stacked[whole, i, : rows - whole * FP8_BLOCK] = t[whole * FP8_BLOCK:]
    return stacked.reshape(2 * runs * FP8_BLOCK, *rest)


__all__ = ["FP8_BLOCK", "Fp8Rows", "Fp8Blocks", "quantize_rows_fp8", "quantize_blocks_fp8", "dequantize_fp8", "add_rmsnorm_fp8", "linear_fp8",
           "gate_up_swiglu_fp8", "stack_gate_up_fp8", "fp8_plan"]
