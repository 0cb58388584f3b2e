"""A dense layer in 8-bit integers: its norms end in int8 rows, and every projection multiplies int8 rows by int8 weights.

Weights are rounded where they are bound, one float32 scale per output feature; activations are rounded token by token on the
way: by the norm in front of a projection, else by a kernel of its own (attention's output, the hidden vector of the
feed-forward).  The residual stream stays float32, attention and its pages stay in the compute dtype, and so do the embedding,
the final norm and the output head.  A layer is then

    norm -> int8 -> q/k/v -> attention -> int8 -> o -> add, norm -> int8 -> gate/up, SwiGLU -> int8 -> down -> (the next norm adds)

The parts are the plain ones with their products replaced; a builder uses them together, since what `Int8RMSNorm` returns only
the other two take.
"""

from __future__ import annotations

import torch

from slipstream_b200 import ops

from .attention import PagedAttention
from .base import FEED_FORWARDS, MIXERS, NORMS, IntoNorm, Runtime
from .mlp import SwiGLUFeedForward
from .norm import RMSNorm


def _as_rows(x: "torch.Tensor | ops.Int8Rows") -> ops.Int8Rows:
    return x if isinstance(x, ops.Int8Rows) else ops.quantize_rows_int8(x, activations=True)


def _close(y: torch.Tensor, into: IntoNorm | None):
    """A branch's output, or the norm of the stream with it added where that was asked for."""
    return y if into is None else into.norm.add_norm(into.residual, y)


@NORMS.register("rmsnorm_int8")
class Int8RMSNorm(RMSNorm):
    """`RMSNorm` whose output is int8 rows, formed from float32 without a rounding in between."""

    def add_norm(self, residual: torch.Tensor, delta: torch.Tensor | None, rows: torch.Tensor | None = None) -> ops.Int8Rows:
        if rows is not None:
            raise ValueError(f"{self.name}: a norm in 8 bits takes every row of the stream")
        return ops.add_rmsnorm_int8(residual, delta, self.weight, self.eps)

    def add_norm_of_linear(self, residual: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None) -> ops.Int8Rows:
        return self.add_norm(residual, ops.linear(x, weight, bias))


@MIXERS.register("paged_attention_int8")
class Int8PagedAttention(PagedAttention):
    """`PagedAttention` with both projections in 8 bits; its input is int8 rows, or a tensor that is rounded here."""

    def bind(self, weights: dict[str, torch.Tensor], runtime: Runtime) -> None:
        super().bind(weights, runtime)
        self.qkv_weight = ops.quantize_rows_int8(self.qkv_weight)
        self.o_weight = ops.quantize_rows_int8(self.o_weight)

    def weight_bytes(self) -> int:
        return self.qkv_weight.nbytes() + self.o_weight.nbytes()

    def project(self, x: "torch.Tensor | ops.Int8Rows") -> torch.Tensor:
        return ops.linear_int8(_as_rows(x), self.qkv_weight, self.qkv_b, self.runtime.dtype)

    def project_out(self, out: torch.Tensor, into: IntoNorm | None):
        return _close(ops.linear_int8(_as_rows(out), self.o_weight, self.o_b, self.runtime.dtype), into)


@FEED_FORWARDS.register("swiglu_int8")
class Int8SwiGLUFeedForward(SwiGLUFeedForward):
    """`SwiGLUFeedForward` with its three products in 8 bits; its input is int8 rows, or a tensor that is rounded here."""

    def bind(self, weights: dict[str, torch.Tensor], runtime: Runtime) -> None:
        if not self.is_swiglu:
            raise ValueError(f"{self.name}: the gated unit in 8 bits is SwiGLU")
        super(SwiGLUFeedForward, self).bind(weights, runtime)
        names = self.names
        self.gate_up = ops.quantize_rows_int8(ops.stack_gate_up(weights[names["gate"]], weights[names["up"]]))
        self.down = ops.quantize_rows_int8(weights[names["down"]])
        self.gate_up_bias = self.down_bias = None
        if self.bias:
            self.gate_up_bias = ops.stack_gate_up(weights[names["gate_bias"]], weights[names["up_bias"]]).to(runtime.dtype)
            self.down_bias = weights[names["down_bias"]].to(runtime.dtype)

    def weight_bytes(self) -> int:
        return self.gate_up.nbytes() + self.down.nbytes()

    def forward(self, x: "torch.Tensor | ops.Int8Rows", ctx, into: IntoNorm | None = None):
        hidden = ops.gate_up_swiglu_int8(_as_rows(x), self.gate_up, self.gate_up_bias, self.runtime.dtype, features=self.intermediate_size)
        return _close(ops.linear_int8(_as_rows(hidden), self.down, self.down_bias, self.runtime.dtype), into)
