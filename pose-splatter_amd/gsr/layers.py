"""Layers of a trainable Gaussian parameter head on libgsr: layer norm and the gated block.

The reference's head is a torch nn.Sequential on [N, channels] voxel features
(src/model.py:207-232); these are the hidden layers of a head on libgsr's kernels, forward and
backward (``gsr.head.GatedHead``; its output projection is a torch.nn.Linear, a library product).
fp32, bf16 and fp16 tensors; arithmetic, sums and statistics are fp32, and gradients are bitwise
deterministic.  Forward-mode derivatives are refused.  No CPU path: the functions raise on CPU
tensors.
"""
from __future__ import annotations

import torch

from ._lib import native

__all__ = ["layer_norm", "LayerNorm", "gated_linear", "GatedLinear", "ACTIVATIONS"]


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over x's last dimension: (x - mean) / sqrt(var + eps) * weight + bias, with the
    biased variance.  x [..., dim]; weight, bias [dim] or None, of x's type or both of another of
    the three (fp32 weights of bf16 features).  Rows of a wider buffer (any row stride) are read
    in place.  Differentiable (once) w.r.t. x, weight and bias."""
    return native().layer_norm(x, weight, bias, eps)


class LayerNorm(torch.nn.Module):
    """``layer_norm`` with its weight and bias as parameters (1 and 0 at first); the parameter
    names and shapes of torch.nn.LayerNorm, so checkpoints of one load into the other."""

    def __init__(self, dim: int, eps: float = 1e-5, bias: bool = True, device=None, dtype=None):
        super().__init__()
        self.dim, self.eps = int(dim), float(eps)
        self.weight = torch.nn.Parameter(torch.ones(self.dim, device=device, dtype=dtype))
        if bias:
            self.bias = torch.nn.Parameter(torch.zeros(self.dim, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"{self.dim}, eps={self.eps}, bias={self.bias is not None}"


ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}   # include/gsr.h GSR_ACT_*


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: torch.Tensor | None = None,
                 b_up: torch.Tensor | None = None, activation: str = "silu") -> torch.Tensor:
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up): both projections, the activation and the
    product in one kernel.  x [..., dim] (any row stride), w_gate and w_up [hidden, dim], the
    biases [hidden] or both None, all of one type; activation "silu", "gelu" (the error
    function's form), "relu" or "sigmoid".  Sums are fp32; in bf16 and fp16 the backward rounds
    the projections' gradients to the type before the products that use them, as separate
    layers would (in small cases and up to 15 columns they stay fp32): a gradient's root mean square
    error is up to 1.4 times that of products of unrounded ones, and in fp16 a projection's gradient
    above 65504 is infinite and one below 2^-25 is zero, so a loss is scaled for them as for any fp16
    layer's.  Differentiable (once) w.r.t. every tensor.  For its backward a forward keeps x and the weights, from dim 256 on (128
    in fp32, where a case is not small) both projections, 6 bytes an element of [rows, hidden] (8
    in fp32), and where dim is not a multiple of 8 (4) a copy of x and the weights that is; below
    that the backward computes the projections again."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"gated_linear: activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    return native().gated_linear(x, w_gate, w_up, b_gate, b_up, act)


class GatedLinear(torch.nn.Module):
    """``gated_linear`` with its weights (and biases) as parameters, initialised as torch.nn.Linear's."""

    def __init__(self, dim: int, hidden: int, activation: str = "silu", bias: bool = True, device=None, dtype=None):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"GatedLinear: activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
        self.dim, self.hidden, self.activation = int(dim), int(hidden), activation
        new = lambda *s: torch.nn.Parameter(torch.empty(*s, device=device, dtype=dtype))  # noqa: E731
        self.w_gate, self.w_up = new(self.hidden, self.dim), new(self.hidden, self.dim)
        if bias:
            self.b_gate, self.b_up = new(self.hidden), new(self.hidden)
        else:
            self.register_parameter("b_gate", None)
            self.register_parameter("b_up", None)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        bound = self.dim ** -0.5
        with torch.no_grad():
            for p in self.parameters():
                p.uniform_(-bound, bound)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return gated_linear(x, self.w_gate, self.w_up, self.b_gate, self.b_up, self.activation)

    def extra_repr(self) -> str:
        return f"{self.dim}, {self.hidden}, activation={self.activation!r}, bias={self.b_gate is not None}"
