"""AdamW on libgsr: one launch steps all tensors, with the moments in 32 or in 8 bits.

The reference trains with torch's Adam (scripts/training/train_script.py:135); next to a render
step of a few milliseconds an optimizer of a dozen launches a tensor is not free, and two fp32
moments of 2 M Gaussian rows are twice the scene itself.

    opt = gsr.optim.AdamW(model.parameters(), lr=1e-3, moment_bits=8)
    (iou_loss + img_loss).backward(); opt.step(); opt.zero_grad()

``adamw_step`` is the step alone, on lists of tensors.  8-bit moments: blocks of 256 elements
(in memory order) with one fp32 unit each; the first moment as float8_e4m3fn codes, the second
as uint8 codes of its root (16 steps a doubling, so that eight bits span the range that the step
needs: the step divides by the root, not by the moment).  Both round to nearest.  The step
itself uses the new moments before they are rounded.  What rounding costs: a root's code moves
once its value has changed by 1/32 relative to its block's largest, so slow changes inside a
block are followed in steps.  No CPU path: the functions raise on CPU tensors.
"""
from __future__ import annotations

import array
import ctypes

import torch

from . import _lib
from ._lib import check, lib
from .layers import _on, _raw_stream, _type
from .render import _require_device

__all__ = ["AdamW", "adamw_step", "decode_root"]

_BLOCK = _lib.ADAMW_BLOCK


def _units(numel: int) -> int:
    return -(-numel // _BLOCK)


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill one stretch of memory, each once, in some order of its dimensions."""
    if t.is_contiguous():
        return True
    n = 1
    for stride, size in sorted((s, d) for s, d in zip(t.stride(), t.shape) if d != 1):
        if stride != n:
            return False
        n *= size
    return True


def _layout(t: torch.Tensor):
    """The strides that matter: those of dimensions of more than one element."""
    return [s for s, d in zip(t.stride(), t.shape) if d != 1]


def _check_layout(t: torch.Tensor, p: torch.Tensor, what: str) -> None:
    if t.shape != p.shape or (_layout(t) != _layout(p) if t.numel() else False):
        raise ValueError(f"adamw_step: {what} must have its parameter's shape and strides {tuple(p.shape)}, "
                         f"{p.stride()}; got {tuple(t.shape)}, {t.stride()}")


def _step_args(lr, betas, eps, weight_decay, step, bits):
    args = _lib.AdamwArgs()
    if isinstance(lr, torch.Tensor):
        if lr.numel() != 1 or lr.dtype != torch.float32:
            raise ValueError("adamw_step: a tensor lr must be one float32 value")
        args.lr, args.lr_dev = 0.0, lr.data_ptr()
    else:
        if not lr >= 0:
            raise ValueError(f"adamw_step: lr must not be negative, got {lr}")
        args.lr, args.lr_dev = float(lr), None
    b1, b2 = betas
    if not (0 <= b1 < 1 and 0 <= b2 < 1):
        raise ValueError(f"adamw_step: betas must be in [0, 1), got {betas}")
    if not (eps >= 0 and weight_decay >= 0):
        raise ValueError(f"adamw_step: eps and weight_decay must not be negative, got {eps}, {weight_decay}")
    args.beta1, args.beta2, args.eps, args.weight_decay = float(b1), float(b2), float(eps), float(weight_decay)
    args.step = 0 if isinstance(step, (torch.Tensor, list, tuple)) else int(step)
    args.bits = bits
    return args


def _no_overlap(ranges) -> None:
    ranges.sort()
    end = 0
    for a, b in ranges:
        if a < end:
            raise ValueError("adamw_step: a tensor is listed twice, or tensors to be written overlap")
        end = b


@torch.no_grad()
def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, step, exp_avg_units=None, exp_avg_root_units=None) -> None:
    """One AdamW step over lists of tensors, in place:

        m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2
        p = p (1 - lr wd) - lr / (1 - b1^step) * m / (sqrt(v) / sqrt(1 - b2^step) + eps)

    params: float32, bfloat16 or float16 tensors on one device that fill their memory (contiguous
    or a permutation of it) and do not overlap; grads of one of these types each.  32-bit moments:
    exp_avgs and exp_avg_sqs are float32, with the parameters' shapes and strides.  8-bit moments
    (when the units are given): exp_avgs are float8_e4m3fn codes, exp_avg_sqs uint8 codes of
    sqrt(v) (``decode_root``), exp_avg_units and exp_avg_root_units float32 [ceil(numel / 256)];
    zeros are zero moments.  lr: a number or one float32 value on the device.  step: the count of
    this step, 1 at first: a number, one int64 value on the device for all tensors, or a list of
    such values; the device forms are read by the kernel (a step captured in a HIP graph)."""
    count = len(params)
    bits = 32 if exp_avg_units is None else 8
    if (exp_avg_units is None) != (exp_avg_root_units is None):
        raise ValueError("adamw_step: exp_avg_units and exp_avg_root_units go together")
    lists = [grads, exp_avgs, exp_avg_sqs] + ([exp_avg_units, exp_avg_root_units] if bits == 8 else [])
    if any(len(x) != count for x in lists):
        raise ValueError(f"adamw_step: {count} params, but lists of {[len(x) for x in lists]}")
    args = _step_args(lr, betas, eps, weight_decay, step, bits)
    if isinstance(step, torch.Tensor):
        step = [step] * count
    steps = list(step) if isinstance(step, (list, tuple)) else None
    if steps is None and args.step < 1:
        raise ValueError(f"adamw_step: step must be at least 1, got {step}")
    if steps is not None and len(steps) != count:
        raise ValueError(f"adamw_step: {count} params, but {len(steps)} steps")
    if count == 0:
        return
    dev = params[0].device
    if args.lr_dev and lr.device != dev:
        raise ValueError(f"adamw_step: lr is on {lr.device}, the parameters on {dev}")
    if bits == 32:
        m_type = v_type = torch.float32
    else:
        m_type, v_type = torch.float8_e4m3fn, torch.uint8
    groups, ranges, kept = {}, [], []
    m_size, v_size = m_type.itemsize, v_type.itemsize
    for i, (p, g, m, v) in enumerate(zip(params, grads, exp_avgs, exp_avg_sqs)):
        if not (p.device == g.device == m.device == v.device == dev):
            raise ValueError(f"adamw_step: tensor {i}, its gradient and moments are on {p.device}, {g.device}, {m.device} "
                             f"and {v.device}; the first tensor is on {dev}")
        types = (p.dtype, g.dtype)
        group = groups.get(types)
        if group is None:
            group = groups[types] = (_type(p, "adamw_step: a parameter"), _type(g, "adamw_step: a gradient"), [])
        if m.dtype != m_type or v.dtype != v_type:
            raise ValueError(f"adamw_step: exp_avg must be {m_type} and exp_avg_sq {v_type}, got {m.dtype} and {v.dtype}")
        if g.layout != torch.strided or g.shape != p.shape:
            raise ValueError(f"adamw_step: gradient {i} must be dense and {tuple(p.shape)}, got {tuple(g.shape)}")
        if not (p.is_contiguous() and g.is_contiguous() and m.is_contiguous() and v.is_contiguous()
                and m.shape == p.shape and v.shape == p.shape):
            if not _dense(p):
                raise ValueError(f"adamw_step: parameter {i} does not fill its memory (strides {p.stride()})")
            _check_layout(m, p, "exp_avg")
            _check_layout(v, p, "exp_avg_sq")
            if _layout(g) != _layout(p):   # (a gradient of another layout: copied into the parameter's)
                g = torch.empty_strided(p.shape, p.stride(), dtype=g.dtype, device=dev).copy_(g)
                kept.append(g)
        n = p.numel()
        if n == 0:
            continue
        pp, mp, vp, mu, vu, sp = p.data_ptr(), m.data_ptr(), v.data_ptr(), 0, 0, 0
        ranges += ((pp, pp + n * p.element_size()), (mp, mp + n * m_size), (vp, vp + n * v_size))
        if bits == 8:
            for u in (exp_avg_units[i], exp_avg_root_units[i]):
                if u.dtype != torch.float32 or u.shape != (_units(n),) or not u.is_contiguous() or u.device != dev:
                    raise ValueError(f"adamw_step: units {i} must be contiguous float32 [{_units(n)}] on {dev}, "
                                     f"got {u.dtype} {tuple(u.shape)} on {u.device}")
            mu, vu = exp_avg_units[i].data_ptr(), exp_avg_root_units[i].data_ptr()
            ranges += ((mu, mu + 4 * _units(n)), (vu, vu + 4 * _units(n)))
        if steps is not None:
            s = steps[i]
            if not isinstance(s, torch.Tensor) or s.numel() != 1 or s.dtype != torch.int64 or s.device != dev:
                raise ValueError(f"adamw_step: step {i} must be one int64 value on {dev}")
            sp = s.data_ptr()
        group[2].extend((pp, g.data_ptr(), mp, vp, mu, vu, sp, n))
    _no_overlap(ranges)
    _require_device(params[0], "adamw_step")
    L = lib()
    with _on(dev):
        stream = _raw_stream(dev)
        for pt, gt, words in groups.values():
            table = array.array("q", words)   # gsr_adamw_tensor: eight 64-bit fields
            check(L.gsr_adamw_step(table.buffer_info()[0], len(words) // 8, pt, gt, ctypes.byref(args), stream),
                  "gsr_adamw_step")
    torch.autograd.graph.increment_version(list(params))


def decode_root(codes: torch.Tensor, units: torch.Tensor) -> torch.Tensor:
    """The roots sqrt(v) (float32, codes' shape) that the uint8 codes of an 8-bit second moment
    stand for; codes contiguous, units [ceil(numel / 256)] float32."""
    if codes.dtype != torch.uint8 or not codes.is_contiguous():
        raise ValueError(f"decode_root: codes must be contiguous uint8, got {codes.dtype}")
    if units.dtype != torch.float32 or units.shape != (_units(codes.numel()),) or not units.is_contiguous() \
            or units.device != codes.device:
        raise ValueError(f"decode_root: units must be contiguous float32 [{_units(codes.numel())}] on {codes.device}, "
                         f"got {units.dtype} {tuple(units.shape)} on {units.device}")
    _require_device(codes, "decode_root")
    out = torch.empty(codes.shape, device=codes.device, dtype=torch.float32)
    with _on(codes.device):
        check(lib().gsr_adamw_decode_root(codes.data_ptr(), units.data_ptr(), codes.numel(), out.data_ptr(),
                                          _raw_stream(codes.device)), "gsr_adamw_decode_root")
    return out


class AdamW(torch.optim.Optimizer):
    """AdamW over ``adamw_step``: torch.optim.AdamW's arguments and update.

    moment_bits 32 or 8: how the moments are held (state "exp_avg", "exp_avg_sq", and with 8 also
    "exp_avg_unit", "exp_avg_root_unit").  capturable=True keeps the step counts on the device, so
    that ``step()`` can be captured in a HIP graph (and takes a float32 device tensor as lr); state
    is then created by one eager step before the capture.  State is float32 or codes whatever the
    parameters' type, also after load_state_dict."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 moment_bits: int = 32, capturable: bool = False):
        if moment_bits not in (8, 32):
            raise ValueError(f"AdamW: moment_bits must be 8 or 32, got {moment_bits}")
        _step_args(lr, betas, eps, weight_decay, 1, moment_bits)   # the same checks as every step's
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      moment_bits=int(moment_bits), capturable=bool(capturable)))

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
            s["exp_avg_unit"] = torch.zeros(_units(p.numel()), device=p.device)
            s["exp_avg_root_unit"] = torch.zeros(_units(p.numel()), device=p.device)
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
                                 exp_avg_root_units=[s["exp_avg_root_unit"] for s in states])
                adamw_step([p for p, _ in items], [p.grad for p, _ in items], [s["exp_avg"] for s in states],
                           [s["exp_avg_sq"] for s in states], lr=group["lr"], betas=group["betas"], eps=group["eps"],
                           weight_decay=group["weight_decay"], step=steps, **units)
                if not group["capturable"]:
                    for s in states:
                        s["step"] = steps
        return loss

    def load_state_dict(self, state_dict: dict) -> None:
        """As torch's, but the moments keep their own types (torch would cast them to the
        parameters')."""
        for mine, saved in zip(self.param_groups, state_dict["param_groups"]):
            if saved.get("moment_bits", 32) != mine["moment_bits"]:
                raise ValueError(f"AdamW: the checkpoint's moments have {saved.get('moment_bits', 32)} bits, "
                                 f"this optimizer's {mine['moment_bits']}")
        super().load_state_dict(state_dict)
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
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
                        to = torch.empty_strided(p.shape, p.stride(), dtype=v.dtype, device=p.device)
                        raw = torch.uint8 if v.element_size() == 1 else v.dtype
                        to.view(raw).copy_(v.to(p.device).view(raw))
                        new[name] = to
                    else:
                        new[name] = v.to(p.device, copy=True)
