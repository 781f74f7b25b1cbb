"""AdamW on libgsr: one launch steps all tensors, with the moments in 32 or in 8 bits.

The reference trains with torch's Adam (scripts/training/train_script.py:135); next to a render
step of a few milliseconds an optimizer of a dozen launches a tensor is not free, and two fp32
moments of 2 M Gaussian rows are twice the scene itself.

    opt = gsr.optim.AdamW(model.parameters(), lr=1e-3, moment_bits=8)
    (iou_loss + img_loss).backward(); opt.step(); opt.zero_grad()

``adamw_step`` is the step alone, on lists of tensors.  8-bit moments: blocks of 256 elements
(in memory order) with one fp32 unit each; the first moment as float8_e4m3fn codes, the second
as uint8 codes of its root (16 steps a doubling, so that eight bits span the range that the step
needs: the step divides by the root, not by the moment).  The step itself uses the new moments
before they are rounded.  ``AdamW`` rounds them up or down without bias, so that over many steps
they follow the moments that are not rounded; one step's rounding is off by less than a code's
step (1/8 of a mean, 1/16 of a root, or a unit).  Rounded to nearest, a change of less than half
a code's step is lost in every step: at beta2 = 0.999 a root would stay where it first was.  No
CPU path: the functions raise on CPU tensors.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import native
from .render import _require_device

__all__ = ["AdamW", "adamw_step", "decode_root"]

_BLOCK = _lib.ADAMW_BLOCK


def _units(numel: int) -> int:
    return -(-numel // _BLOCK)


def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one shape order their elements in memory alike."""
    return a.numel() == 0 or all(n == 1 or x == y for n, x, y in zip(a.shape, a.stride(), b.stride()))


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, step, exp_avg_units=None, exp_avg_root_units=None,
               moment_rounding: str = "nearest") -> None:
    """One AdamW step over lists of tensors, in place:

        m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2
        p = p (1 - lr wd) - lr / (1 - b1^step) * m / (sqrt(v) / sqrt(1 - b2^step) + eps)

    params: float32, bfloat16 or float16 tensors on one device that fill their memory (contiguous
    or a permutation of it) and do not overlap; grads of one of these types each.  32-bit moments:
    exp_avgs and exp_avg_sqs are float32, with the parameters' shapes and strides.  8-bit moments
    (when the units are given): exp_avgs are float8_e4m3fn codes, exp_avg_sqs uint8 codes of
    sqrt(v) (``decode_root``), exp_avg_units and exp_avg_root_units float32 [ceil(numel / 256)];
    zeros are zero moments.  moment_rounding, of 8-bit moments: "nearest" (ties to even; a change of
    less than half a code's step is lost, so this is for single steps and conversions), or
    "unbiased": up with the probability that keeps the expected m and v, drawn by a hash of the element's
    place in its tensor and the step count (the same bits every run, in any list).  A root below
    one unit (1/507904 of its block's largest) is held as one in both.  lr: a number or one float32 value on the device.  step: the count of
    this step, 1 at first: a number, one int64 value on the device for all tensors, or a list of
    such values; the device forms are read by the kernel (a step captured in a HIP graph)."""
    lr_dev = lr if isinstance(lr, torch.Tensor) else None
    if isinstance(step, torch.Tensor):
        step = [step] * len(params)
    steps = step if isinstance(step, (list, tuple)) else None
    if moment_rounding not in ("nearest", "unbiased"):
        raise ValueError(f'adamw_step: moment_rounding must be "nearest" or "unbiased", got {moment_rounding!r}')
    native().adamw_step(params, grads, exp_avgs, exp_avg_sqs, 0.0 if lr_dev is not None else lr, lr_dev, *betas, eps,
                        weight_decay, 0 if steps is not None else step, steps, exp_avg_units, exp_avg_root_units,
                        moment_rounding == "unbiased")


def decode_root(codes: torch.Tensor, units: torch.Tensor) -> torch.Tensor:
    """The roots sqrt(v) (float32, codes' shape) that the uint8 codes of an 8-bit second moment
    stand for; codes contiguous, units [ceil(numel / 256)] float32."""
    return native().decode_root(codes, units)


class AdamW(torch.optim.Optimizer):
    """AdamW over ``adamw_step``: torch.optim.AdamW's arguments and update.

    moment_bits 32 or 8: how the moments are held (state "exp_avg", "exp_avg_sq", and with 8 also
    "exp_avg_unit", "exp_avg_root_unit"); 8-bit ones are rounded without bias.  capturable=True keeps the step counts on the device, so
    that ``step()`` can be captured in a HIP graph (and takes a float32 device tensor as lr); state
    is then created by one eager step before the capture.  State is float32 or codes whatever the
    parameters' type, also after load_state_dict."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 moment_bits: int = 32, capturable: bool = False):
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      moment_bits=moment_bits, capturable=bool(capturable)))

    def add_param_group(self, param_group: dict) -> None:
        """As torch's; a group's own values are checked like the defaults."""
        super().add_param_group(param_group)
        try:
            self._check_group(self.param_groups[-1])
        except (ValueError, TypeError):
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_group(g: dict) -> None:
        if g["moment_bits"] not in (8, 32):
            raise ValueError(f"AdamW: moment_bits must be 8 or 32, got {g['moment_bits']}")
        adamw_step([], [], [], [], lr=g["lr"], betas=g["betas"], eps=g["eps"], weight_decay=g["weight_decay"], step=1)

    def _state(self, p: torch.Tensor, group: dict) -> dict:
        s = self.state[p]
        if s:
            return s
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: take one eager step before capturing (it creates the moments)")
        like = dict(size=p.shape, stride=p.stride(), device=p.device)
        if group["moment_bits"] == 32:
            s["exp_avg"] = torch.empty_strided(**like, dtype=torch.float32).zero_()
            s["exp_avg_sq"] = torch.empty_strided(**like, dtype=torch.float32).zero_()
        else:
            s["exp_avg"] = torch.empty_strided(**like, dtype=torch.uint8).zero_().view(torch.float8_e4m3fn)
            s["exp_avg_sq"] = torch.empty_strided(**like, dtype=torch.uint8).zero_()
            s["exp_avg_unit"] = torch.zeros(_units(p.numel()), device=p.device, dtype=torch.float32)
            s["exp_avg_root_unit"] = torch.zeros(_units(p.numel()), device=p.device, dtype=torch.float32)
        s["step"] = torch.zeros((), dtype=torch.int64, device=p.device) if group["capturable"] else 0
        return s

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            if not group["capturable"] and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: a captured step would repeat one step count; use capturable=True")
            buckets = {}   # (device, host step count): tensors stepped together
            for p in group["params"]:
                if p.grad is None:
                    continue
                _require_device(p, "AdamW")
                if p.grad.is_sparse or p.is_complex():
                    raise ValueError("AdamW: sparse gradients and complex parameters are not supported")
                s = self._state(p, group)
                key = (p.device, None if group["capturable"] else s["step"])
                buckets.setdefault(key, []).append((p, s))
            for (_, count), items in buckets.items():
                states = [s for _, s in items]
                if group["capturable"]:
                    steps = [s["step"] for s in states]
                    torch._foreach_add_(steps, 1)
                else:
                    steps = count + 1
                units = {}
                if group["moment_bits"] == 8:
                    units = dict(exp_avg_units=[s["exp_avg_unit"] for s in states],
                                 exp_avg_root_units=[s["exp_avg_root_unit"] for s in states], moment_rounding="unbiased")
                try:
                    adamw_step([p for p, _ in items], [p.grad for p, _ in items], [s["exp_avg"] for s in states],
                               [s["exp_avg_sq"] for s in states], lr=group["lr"], betas=group["betas"], eps=group["eps"],
                               weight_decay=group["weight_decay"], step=steps, **units)
                except Exception:
                    if group["capturable"]:   # (a refused step was none)
                        torch._foreach_sub_(steps, 1)
                    raise
                if not group["capturable"]:
                    for s in states:
                        s["step"] = steps
        return loss

    def load_state_dict(self, state_dict: dict) -> None:
        """As torch's, but the moments keep their own types (torch would cast them to the
        parameters').  8-bit moments are taken only by a parameter of their own memory order (their
        units belong to runs of 256 elements in that order); 32-bit ones follow the parameter's.
        A torch.optim.AdamW checkpoint is taken too, its moments as float32, unless its update is
        another one (amsgrad, maximize, decay in the gradient)."""
        options = [{k: g[k] for k in ("moment_bits", "capturable")} for g in self.param_groups]
        final = {}   # what the caller's own hooks leave of state_dict

        def check(_, sd):
            for mine, saved in zip(self.param_groups, sd["param_groups"]):
                self._check_saved(mine, saved, sd["state"])
            final.update(sd)

        hooks = [self.register_load_state_dict_pre_hook(check),   # after the caller's, the next before
                 self.register_load_state_dict_post_hook(lambda _: self._take(final, options), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for h in hooks:
                h.remove()

    def _take(self, state_dict: dict, options: list) -> None:
        for group, saved, own in zip(self.param_groups, state_dict["param_groups"], options):
            for k, v in own.items():
                group.setdefault(k, v)
            if isinstance(group["lr"], torch.Tensor) and group["params"]:
                group["lr"] = group["lr"].to(group["params"][0].device, torch.float32)
            for p, key in zip(group["params"], saved["params"]):
                s = state_dict["state"].get(key)
                if not s:
                    continue
                new = self.state[p] = {}
                for name, v in s.items():
                    if name == "step":
                        new[name] = (torch.tensor(int(v), dtype=torch.int64, device=p.device) if group["capturable"]
                                     else int(v))
                    elif name in ("exp_avg", "exp_avg_sq"):
                        v = v.to(p.device, torch.float32 if group["moment_bits"] == 32 else v.dtype)
                        to = torch.empty_strided(p.shape, p.stride(), dtype=v.dtype, device=p.device)
                        raw = torch.uint8 if v.element_size() == 1 else v.dtype
                        to.view(raw).copy_(v.view(raw))
                        new[name] = to
                    else:
                        new[name] = v.to(p.device, copy=True)

    def _check_saved(self, mine: dict, saved: dict, state: dict) -> None:
        if saved.get("moment_bits", 32) != mine["moment_bits"]:
            raise ValueError(f"AdamW: the checkpoint's moments have {saved.get('moment_bits', 32)} bits, "
                             f"this optimizer's {mine['moment_bits']}")
        for option in ("amsgrad", "maximize"):
            if saved.get(option):
                raise ValueError(f"AdamW: the checkpoint's steps are taken with {option}=True, which this optimizer has not")
        if not saved.get("decoupled_weight_decay", True) and saved["weight_decay"] != 0:
            raise ValueError("AdamW: the checkpoint's weight decay is part of the gradient, this optimizer's is decoupled")
        lr = saved["lr"]
        self._check_group({**mine, **saved, "lr": lr.float() if isinstance(lr, torch.Tensor) else lr})
        for p, key in zip(mine["params"], saved["params"]):
            s = state.get(key)
            if not s:
                continue
            if any(s[k].shape != p.shape for k in ("exp_avg", "exp_avg_sq")):
                raise ValueError(f"AdamW: the checkpoint's moments of parameter {key} have the shape "
                                 f"{tuple(s['exp_avg'].shape)}, the parameter {tuple(p.shape)}")
            if mine["moment_bits"] == 8 and not all(_same_order(s[k], p) for k in ("exp_avg", "exp_avg_sq")):
                raise ValueError(f"AdamW: the checkpoint's 8-bit moments of parameter {key} have strides "
                                 f"{s['exp_avg'].stride()}, another memory order than the parameter's {p.stride()}: load "
                                 "them into a parameter of their order")
