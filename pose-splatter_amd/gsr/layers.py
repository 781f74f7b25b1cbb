"""Layers of a trainable Gaussian parameter head on libgsr: layer norm.

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
from .render import _ptr, _require_device, _stream

__all__ = ["layer_norm", "LayerNorm"]

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


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        L = lib()
        dim = x.shape[-1]
        xr, stride = _as_rows(x, dim)
        rows = xr.shape[0]
        y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        need = any(ctx.needs_input_grad[:3])
        stats = torch.empty(rows, 2, device=x.device, dtype=torch.float32) if need else None
        wt = _TYPE[(weight if weight is not None else bias if bias is not None else x).dtype]
        with _on(x.device):
            check(L.gsr_layer_norm_fwd(_ptr(xr), rows, dim, stride, _TYPE[x.dtype], _ptr(weight), _ptr(bias), wt, eps,
                                       _ptr(y), _ptr(stats), _stream(x.device)), "gsr_layer_norm_fwd")
        if need:
            ctx.save_for_backward(xr, weight, stats)
            ctx.cfg = (x.shape, stride, wt, bias is not None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        L = lib()
        xr, weight, stats = ctx.saved_tensors
        shape, stride, wt, has_bias = ctx.cfg
        rows, dim = xr.shape
        if g.dtype != xr.dtype:
            g = g.to(xr.dtype)
        g, g_stride = _as_rows(g, dim)
        dev = xr.device
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        like = {_lib.F32: torch.float32, _lib.BF16: torch.bfloat16, _lib.F16: torch.float16}[wt]
        dx = torch.empty(shape, device=dev, dtype=xr.dtype) if need_x else None
        dw = torch.empty(dim, device=dev, dtype=like) if need_w else None
        db = torch.empty(dim, device=dev, dtype=like) if need_b and has_bias else None
        ws = None
        if dw is not None or db is not None:
            ws = torch.empty(int(L.gsr_layer_norm_workspace(rows, dim, _TYPE[xr.dtype])), device=dev, dtype=torch.uint8)
        with _on(dev):
            check(L.gsr_layer_norm_bwd(_ptr(xr), _ptr(g), rows, dim, stride, g_stride, _TYPE[xr.dtype], _ptr(weight), wt,
                                       _ptr(stats), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws),
                                       0 if ws is None else ws.numel(), _stream(dev)), "gsr_layer_norm_bwd")
        return dx, dw, db, None


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
