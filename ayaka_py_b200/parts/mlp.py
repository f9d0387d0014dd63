"""Dense feed-forward: up projection, activation, down projection, residual
(``models/gpt2.py:400-403``, ``:437-438``).  Bias, activation (in 32-bit) and
the residual sum are fused into the two matrix products' epilogues.

``weight_bits`` 4: the weights are rounded to 4 bits when they are bound (``microscale``), the rows that meet them are 8-bit.  What is
bound has the compute dtype: float32 weights of a bfloat16 model are rounded twice, which gives 1.4 % of the bytes (two codes each) another value than
one rounding would."""

from __future__ import annotations

import torch

from .. import ops
from ..microscale import BLOCK, matrix4
from .base import FeedForward, NotLowered, TensorDecl, register_part
from .stacked import StackedInput


def _check_bits(weight_bits: int, activation: str, *widths: int) -> int:
    if weight_bits not in (4, 16):
        raise ValueError(f"weight_bits must be 16 (the compute dtype) or 4, got {weight_bits!r}")
    if weight_bits == 4 and any(w % BLOCK for w in widths):
        raise ValueError(f"4-bit weights come in blocks of {BLOCK}: widths {widths}")
    if weight_bits == 4 and activation not in ops.ACTIVATIONS:
        raise ValueError(f"no activation {activation!r} with 4-bit weights; known: {sorted(ops.ACTIVATIONS)}")
    return weight_bits


class MLP(FeedForward):
    KIND = "mlp"

    def __init__(self, width: int, inner: int, activation: str, bias: bool = True,
                 dtype=torch.float32, device="cuda", weight_bits: int = 16):
        if activation not in ops.ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}; known: {sorted(ops.ACTIVATIONS)}")
        self.width, self.inner, self.activation, self.has_bias = width, inner, activation, bias
        self.dtype = dtype
        self.weight_bits = _check_bits(weight_bits, activation, width, inner)
        self.up_weight = self.up_bias = self.down_weight = self.down_bias = self.up4 = self.down4 = None

    def tensors(self):
        out = {"up_weight": TensorDecl((self.inner, self.width), "matrix"),
               "down_weight": TensorDecl((self.width, self.inner), "matrix")}
        if self.has_bias:
            out["up_bias"] = TensorDecl((self.inner,), "vector")
            out["down_bias"] = TensorDecl((self.width,), "vector")
        return out

    def bind(self, tensors):
        super().bind(tensors)
        if self.weight_bits == 4:
            self.up4, self.down4 = matrix4(self.up_weight), matrix4(self.down_weight)
            self.up_weight = self.down_weight = None

    def laid_out(self):
        return [t for m in (self.up4, self.down4) if m is not None for t in (m.codes, m.scales)]

    def forward(self, h, residual, ctx):
        if self.weight_bits == 4:
            u = ops.linear4(ops.rows8(h), self.up4, self.up_bias, self.activation, out_dtype=self.dtype)
            return ops.linear4(ops.rows8(u), self.down4, self.down_bias, residual=residual, out_dtype=torch.float32, out=residual)
        u = ops.linear(h, self.up_weight, self.up_bias, activation=self.activation, out_dtype=self.dtype)
        return ops.linear(u, self.down_weight, self.down_bias, residual=residual,
                          out_dtype=torch.float32, out=residual)

    def lower(self, builder, h, residual):
        if self.weight_bits == 4:
            raise NotLowered(type(self).__name__)
        u = builder.linear(h, self.up_weight, self.up_bias, activation=self.activation, out_dtype=self.dtype)
        out = builder.linear(u, self.down_weight, self.down_bias, residual=residual, out_dtype=torch.float32, out=residual)
        builder.release(u)
        return out


class PolyNormMLP(FeedForward):
    """down(act(up h)) without biases, act = PolyNorm: a N(z) + b N(z^2) + c N(z^3) + e with powers
    taken element by element and N the division of a token's vector by its root mean square
    (eps inside the root); the four numbers are a tensor of the part.  The up projection is
    stored in 32-bit, the norms are 32-bit, the activation is stored in the compute dtype."""

    KIND = "polynorm_mlp"

    def __init__(self, width: int, inner: int, eps: float, dtype=torch.float32, device="cuda"):
        self.width, self.inner, self.eps, self.dtype = width, inner, float(eps), dtype
        self.up_weight = self.down_weight = self.coeff = None

    def tensors(self):
        return {"up_weight": TensorDecl((self.inner, self.width), "matrix"),
                "down_weight": TensorDecl((self.width, self.inner), "matrix"),
                "coeff": TensorDecl((4,), "vector")}

    def forward(self, h, residual, ctx):
        """residual + ff(h); with ``residual`` None the sublayer's output alone, float32."""
        z = ops.linear(h, self.up_weight, None, out_dtype=torch.float32)
        u = ops.polynorm(z, self.coeff, self.eps, self.dtype)
        return ops.linear(u, self.down_weight, None, residual=residual, out_dtype=torch.float32, out=residual)


class GatedMLP(FeedForward):
    """down(act(gate h) * (up h)) without biases.  gate | up is one product, stored in 32-bit; the
    activation and the product of the halves are 32-bit, their result is stored in the compute dtype.
    ``activation`` "limited_glu": g sigmoid(slope g) (u + plus) with g = min(gate h, limit) and
    u = clamp(up h, -limit, limit) instead."""

    KIND = "gated_mlp"

    def __init__(self, width: int, inner: int, activation: str, limit: float | None = None, slope: float = 1.702, plus: float = 1.0,
                 dtype=torch.float32, device="cuda", weight_bits: int = 16):
        if activation != "limited_glu" and activation not in ops.ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}; known: {sorted(ops.ACTIVATIONS)} and 'limited_glu'")
        self.width, self.inner, self.activation, self.dtype = width, inner, activation, dtype
        self.limit, self.slope, self.plus = float("inf") if limit is None else float(limit), float(slope), float(plus)
        self.weight_bits = _check_bits(weight_bits, activation, width, inner)
        self.gate_weight = self.up_weight = self.down_weight = self.stack = self.joined = self.matrices = None

    def tensors(self):
        return {"gate_weight": TensorDecl((self.inner, self.width), "matrix"),
                "up_weight": TensorDecl((self.inner, self.width), "matrix"),
                "down_weight": TensorDecl((self.width, self.inner), "matrix")}

    def bind(self, tensors):
        super().bind(tensors)
        if self.weight_bits == 4:
            self.matrices = [matrix4(w) for w in (self.gate_weight, self.up_weight, self.down_weight)]
            self.gate_weight = self.up_weight = self.down_weight = None
            return
        self.stack = StackedInput(self.width, [[self.gate_weight, self.up_weight]])
        self.gate_weight, self.up_weight = self.stack.views[:2]

    def laid_out(self):
        return [t for m in self.matrices or () for t in (m.codes, m.scales)]

    @property
    def in_weight(self):
        """gate | up in one matrix (None where the weights are 4-bit)."""
        return None if self.weight_bits == 4 else self.stack.weight

    def join_input(self, weight, bias):
        if self.weight_bits == 4:
            return None
        at = self.stack.join(weight, bias)
        self.gate_weight, self.up_weight = self.stack.views[:2]
        self.joined = (at, at + weight.shape[0])
        return self.stack.views[-1]

    def forward(self, h, residual, ctx):
        """residual + ff(h); with ``residual`` None the sublayer's output alone, float32."""
        if self.weight_bits == 4:
            gate, up, down = self.matrices
            u = ops.gated_linear4(ops.rows8(h), gate, up, self.activation)
            return ops.linear4(u, down, residual=residual, out_dtype=torch.float32, out=residual)
        z = ops.linear(h, self.stack.weight, self.stack.bias, out_dtype=torch.float32)
        if self.joined is not None:
            ctx.carry[self] = z[:, self.joined[0]:self.joined[1]]
        if self.activation == "limited_glu":
            u = ops.glu_limited(z, self.inner, self.limit, self.slope, self.dtype, self.plus)
        else:
            u = ops.gated_act(z, self.inner, self.activation, self.dtype)
        return ops.linear(u, self.down_weight, None, residual=residual, out_dtype=torch.float32, out=residual)


register_part(MLP.KIND, MLP)
register_part(GatedMLP.KIND, GatedMLP)
register_part(PolyNormMLP.KIND, PolyNormMLP)
