"""Layers of a trainable Gaussian parameter head on libgsr: layer norm and the gated block.

The reference's head is a torch nn.Sequential on [N, channels] voxel features
(src/model.py:207-232); these are the layers of a head that stays on libgsr's kernels from the
features to the renderer rows, forward and backward (``gsr.head.GatedHead``).  fp32, bf16 and
fp16 tensors; arithmetic, sums and statistics are fp32, and gradients are bitwise deterministic.
No CPU path: the functions raise on CPU tensors.
"""
from __future__ import annotations

import contextlib

import torch

from . import _lib
from ._lib import check, lib
from .render import _ptr, _require_device

__all__ = ["layer_norm", "LayerNorm", "gated_linear", "GatedLinear", "ACTIVATIONS"]

_TYPE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _type(t: torch.Tensor, what: str) -> int:
    code = _TYPE.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


_here = contextlib.nullcontext()


def _on(device: torch.device):
    """A context in which ``device``, where a launch goes, is the current one."""
    return _here if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _same_device(x: torch.Tensor, who: str, **others) -> None:
    for name, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{who}: {name} is on {t.device}, the input on {x.device}")


def _as_rows(x: torch.Tensor, dim: int) -> tuple[torch.Tensor, int]:
    """(x as [rows, dim] with unit stride inside a row, its row stride): a view where x is one
    matrix of evenly spaced rows, else a copy."""
    if x.dim() != 2:
        x = x.reshape(-1, dim)
    rows = x.shape[0]
    if (dim > 1 and x.stride(1) != 1) or (rows > 1 and x.stride(0) < dim):
        x = x.contiguous()
    return x, x.stride(0) if rows > 1 else dim


_DTYPE = {code: dtype for dtype, code in _TYPE.items()}


def _raw_stream(device: torch.device) -> int:
    """``_stream`` without its Python wrapper objects (small calls are bound by the host)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        L = lib()
        dev, dim, xt = x.device, x.shape[-1], _TYPE[x.dtype]
        xr, stride = _as_rows(x, dim)
        rows = xr.shape[0]
        y = torch.empty(x.shape, device=dev, dtype=x.dtype)
        need = any(ctx.needs_input_grad)
        stats = torch.empty(rows, 2, device=dev, dtype=torch.float32) if need else None
        wt = _TYPE[(weight if weight is not None else bias if bias is not None else x).dtype]
        with _on(dev):
            check(L.gsr_layer_norm_fwd(xr.data_ptr(), rows, dim, stride, xt, _ptr(weight), _ptr(bias), wt, eps,
                                       y.data_ptr(), _ptr(stats), _raw_stream(dev)), "gsr_layer_norm_fwd")
        if need:
            ctx.save_for_backward(xr, weight, stats)
            ctx.cfg = (x.shape, stride, xt, wt)
        return y

    @staticmethod
    def backward(ctx, g):
        return (_once if torch.is_grad_enabled() else _direct)(_LayerNorm._gradients, ctx, g)

    @staticmethod
    def _gradients(ctx, g):
        L = lib()
        xr, weight, stats = ctx.saved_tensors
        shape, stride, xt, wt = ctx.cfg
        dev = xr.device
        rows, dim = xr.shape
        g, g_stride = _as_rows(g if g.dtype == xr.dtype else g.to(xr.dtype), dim)
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        dx = torch.empty(shape, device=dev, dtype=xr.dtype) if need_x else None
        dw = torch.empty(dim, device=dev, dtype=_DTYPE[wt]) if need_w else None
        db = torch.empty(dim, device=dev, dtype=_DTYPE[wt]) if need_b else None
        ws, ws_bytes = None, 0
        if need_w or need_b:
            ws_bytes = L.gsr_layer_norm_workspace(rows, dim, xt)
            ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
        with _on(dev):
            check(L.gsr_layer_norm_bwd(xr.data_ptr(), g.data_ptr(), rows, dim, stride, g_stride, xt, _ptr(weight), wt,
                                       stats.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), ws_bytes,
                                       _raw_stream(dev)), "gsr_layer_norm_bwd")
        return dx, dw, db, None


def _direct(f, ctx, g):
    return f(ctx, g)


@torch.autograd.function.once_differentiable
def _refuse_twice(ctx, f, g):
    return f(ctx, g)


def _once(f, ctx, g):
    """Under create_graph=True: gradients whose own backward raises (the kernels are differentiable once)."""
    return _refuse_twice(ctx, f, g)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over x's last dimension: (x - mean) / sqrt(var + eps) * weight + bias, with the
    biased variance.  x [..., dim]; weight, bias [dim] or None, of x's type or both of another of
    the three (fp32 weights of bf16 features).  Rows of a wider buffer (any row stride) are read
    in place.  Differentiable (once) w.r.t. x, weight and bias."""
    _type(x, "layer_norm: x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: x must be [..., dim] with dim >= 1, got {tuple(x.shape)}")
    dim = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _type(t, f"layer_norm: {name}")
            if t.shape != (dim,):
                raise ValueError(f"layer_norm: {name} must be [{dim}], got {tuple(t.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"layer_norm: weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps must not be negative, got {eps}")
    _same_device(x, "layer_norm", weight=weight, bias=bias)
    _require_device(x, "layer_norm")
    weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    bias = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    return _LayerNorm.apply(x, weight, bias, float(eps))


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


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        L = lib()
        dev, dim, hidden, t = x.device, x.shape[-1], w_gate.shape[0], _TYPE[x.dtype]
        xr, stride = _as_rows(x, dim)
        h = torch.empty((*x.shape[:-1], hidden), device=dev, dtype=x.dtype)
        ws_bytes = L.gsr_gated_workspace(xr.shape[0], dim, hidden, t, 0)
        ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8) if ws_bytes else None
        with _on(dev):
            check(L.gsr_gated_fwd(xr.data_ptr(), xr.shape[0], dim, stride, t, w_gate.data_ptr(), w_up.data_ptr(), hidden,
                                  _ptr(b_gate), _ptr(b_up), act, h.data_ptr(), _ptr(ws), ws_bytes, _raw_stream(dev)),
                  "gsr_gated_fwd")
        if any(ctx.needs_input_grad):
            ctx.save_for_backward(xr, w_gate, w_up, b_gate, b_up)
            ctx.cfg = (x.shape, stride, t, act)
        return h

    @staticmethod
    def backward(ctx, g):
        return (_once if torch.is_grad_enabled() else _direct)(_GatedLinear._gradients, ctx, g)

    @staticmethod
    def _gradients(ctx, g):
        L = lib()
        xr, wg, wu, bg, bu = ctx.saved_tensors
        shape, stride, t, act = ctx.cfg
        dev, dtype = xr.device, xr.dtype
        rows, dim = xr.shape
        hidden = wg.shape[0]
        g, g_stride = _as_rows(g if g.dtype == dtype else g.to(dtype), hidden)
        sizes = (shape, wg.shape, wu.shape, (hidden,), (hidden,))
        grads = [torch.empty(s, device=dev, dtype=dtype) if need else None
                 for s, need in zip(sizes, ctx.needs_input_grad)]
        ws_bytes = L.gsr_gated_workspace(rows, dim, hidden, t, 1)
        ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
        with _on(dev):
            check(L.gsr_gated_bwd(xr.data_ptr(), rows, dim, stride, t, wg.data_ptr(), wu.data_ptr(), hidden, _ptr(bg),
                                  _ptr(bu), act, g.data_ptr(), g_stride, *map(_ptr, grads), ws.data_ptr(), ws_bytes,
                                  _raw_stream(dev)), "gsr_gated_bwd")
        return (*grads, None)


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: torch.Tensor | None = None,
                 b_up: torch.Tensor | None = None, activation: str = "silu") -> torch.Tensor:
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up): both projections, the activation and the
    product in one kernel.  x [..., dim] (any row stride), w_gate and w_up [hidden, dim], the
    biases [hidden] or both None, all of one type; activation "silu", "gelu" (the error
    function's form), "relu" or "sigmoid".  Sums are fp32; in bf16 and fp16 the backward rounds
    the projections' gradients to the type before the products that use them, as separate
    layers would.  Differentiable (once) w.r.t. every tensor; the backward keeps no
    [rows, hidden] tensor from the forward but computes both projections again."""
    _type(x, "gated_linear: x")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"gated_linear: activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"gated_linear: x must be [..., dim] with dim >= 1, got {tuple(x.shape)}")
    if w_gate.dim() != 2 or w_gate.shape[1] != x.shape[-1] or w_gate.shape[0] < 1 or w_up.shape != w_gate.shape:
        raise ValueError(f"gated_linear: w_gate and w_up must be [hidden, {x.shape[-1]}], got {tuple(w_gate.shape)} and "
                         f"{tuple(w_up.shape)}")
    if (b_gate is None) != (b_up is None):
        raise ValueError("gated_linear: b_gate and b_up go together")
    if b_gate is not None and (b_gate.shape != w_gate.shape[:1] or b_up.shape != w_gate.shape[:1]):
        raise ValueError(f"gated_linear: the biases must be [{w_gate.shape[0]}], got {tuple(b_gate.shape)} and "
                         f"{tuple(b_up.shape)}")
    others = (w_gate, w_up) if b_gate is None else (w_gate, w_up, b_gate, b_up)
    for t in others:
        if t.dtype != x.dtype:
            raise ValueError(f"gated_linear: weights and biases must have x's type {x.dtype}, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"gated_linear: a weight or bias is on {t.device}, x on {x.device}")
    if max(w_gate.shape) > 1 << 20 or x.numel() > x.shape[-1] << 26:
        raise ValueError(f"gated_linear: at most 2^26 rows and 2^20 columns, got {tuple(x.shape)}, {tuple(w_gate.shape)}")
    _require_device(x, "gated_linear")
    w_gate, w_up = w_gate.contiguous(), w_up.contiguous()
    if b_gate is not None:
        b_gate, b_up = b_gate.contiguous(), b_up.contiguous()
    return _GatedLinear.apply(x, w_gate, w_up, b_gate, b_up, act)


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
