"""Group norm with an activation (and dropout) in the same pass, channels last, and its interval form.

Beside the mean shift (MeanNorm, BoundMeanNorm): where a net needs the spread of its activations normalised as well, per sample,
so that evaluation and training compute the same.  A group norm is not 1-Lipschitz in the sup norm as a distance layer is: its
place is the head behind the distance layers, and a certificate takes its bounds from `group_norm_bound`.
zbh2047/L_inf-dist-net has no counterpart.  Kernels: csrc/group_norm.cu, csrc/group_norm_bound.cu.
"""
import math

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib
from .dropout import DropoutF, _Masks, _TYPES, _floating, _generator_state, _rate, dropout_next
from .norm_dist import _on, _scratch, _stream, skips_values

ACTIVATIONS = {"identity": 0, "relu": 1, "tanh": 2, "silu": 3}        # LINF_ACT_*


def _rows(t):
    """[N, C, ...] -> its memory as [N, ..., C]: the tensor itself where the channels lie last, or a copy."""
    t = t.movedim(1, -1)
    return t if t.is_contiguous() else t.contiguous()


def _empty(shape, like):
    """[N, C, ...] with the channels last in memory."""
    if len(shape) == 2:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    strides, step = [0] * len(shape), shape[1]
    strides[1] = 1
    for k in range(len(shape) - 1, 1, -1):
        strides[k] = step
        step *= shape[k]
    strides[0] = step
    return torch.empty_strided(shape, strides, dtype=like.dtype, device=like.device)


def _sizes(shape, groups):
    return shape[0], shape[1], groups, math.prod(shape[2:])


def _ptr(t):
    return None if t is None else t.data_ptr()


class GroupNormF(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, rate, rng):
        lib = _lib.load()
        rows = _rows(x)
        y = _empty(x.shape, x)
        sizes = _sizes(x.shape, groups)
        kept = any(ctx.needs_input_grad[:3])
        stats = torch.empty((2, sizes[0], groups) if kept else (0,), device=x.device, dtype=torch.float32)
        ctx.call = (sizes, _TYPES[x.dtype], _TYPES[weight.dtype] if weight is not None else _TYPES[bias.dtype] if bias is not None else 0, act, rate)
        if x.numel() > 0:
            with _on(x.device):
                need = lib.linf_group_norm_workspace_bytes(*sizes, ctx.call[1], 0)
                ws = _scratch(x.device, need)
                rc = lib.linf_group_norm_forward(rows.data_ptr(), _ptr(weight), _ptr(bias), *sizes, *ctx.call[1:3], eps, act, rate, _ptr(rng),
                                                 y.data_ptr(), stats[0].data_ptr() if kept else None, stats[1].data_ptr() if kept else None,
                                                 ws.data_ptr(), need, _stream())
            _lib.check(rc, "group_norm_forward")
        if kept:
            ctx.save_for_backward(rows, weight, bias, stats, rng)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        lib = _lib.load()
        rows, weight, bias, stats, rng = ctx.saved_tensors
        sizes, kind, ptype, act, rate = ctx.call
        g = _rows(grad_output)
        gx = _empty(grad_output.shape, rows) if ctx.needs_input_grad[0] else None
        gw = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        gb = torch.empty_like(bias) if ctx.needs_input_grad[2] else None
        if rows.numel() == 0:
            return gx, gw if gw is None else gw.zero_(), gb if gb is None else gb.zero_(), None, None, None, None, None
        with _on(rows.device):
            need = lib.linf_group_norm_workspace_bytes(*sizes, kind, 1)
            ws = _scratch(rows.device, need)
            rc = lib.linf_group_norm_backward(g.data_ptr(), rows.data_ptr(), _ptr(weight), _ptr(bias), stats[0].data_ptr(), stats[1].data_ptr(),
                                              *sizes, kind, ptype, act, rate, _ptr(rng), _ptr(gx), _ptr(gw), _ptr(gb), ws.data_ptr(), need, _stream())
        _lib.check(rc, "group_norm_backward")
        return gx, gw, gb, None, None, None, None, None


class GroupNormBoundF(torch.autograd.Function):

    @staticmethod
    def forward(ctx, lower, upper, weight, bias, groups, eps, act):
        lib = _lib.load()
        l, u = _rows(lower), _rows(upper)
        lo, up = _empty(lower.shape, lower), _empty(lower.shape, lower)
        sizes = _sizes(lower.shape, groups)
        kept = any(ctx.needs_input_grad[:4])
        sums = torch.empty((sizes[0], groups, 4) if kept else (0,), device=lower.device, dtype=torch.float64)
        ctx.call = (sizes, eps, act)
        if lower.numel() > 0:
            with _on(lower.device):
                need = lib.linf_group_norm_bound_workspace_bytes(*sizes, 0)
                ws = _scratch(lower.device, need)
                rc = lib.linf_group_norm_bound_forward(l.data_ptr(), u.data_ptr(), _ptr(weight), _ptr(bias), *sizes, eps, act, lo.data_ptr(),
                                                       up.data_ptr(), sums.data_ptr() if kept else None, ws.data_ptr(), need, _stream())
            _lib.check(rc, "group_norm_bound_forward")
        if kept:
            ctx.save_for_backward(l, u, weight, bias, sums)
        return lo, up

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_lower, grad_upper):
        lib = _lib.load()
        l, u, weight, bias, sums = ctx.saved_tensors
        sizes, eps, act = ctx.call
        gl, gu = _rows(grad_lower), _rows(grad_upper)
        box = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        dl, du = (_empty(grad_lower.shape, l), _empty(grad_lower.shape, l)) if box else (None, None)
        gw = torch.empty_like(weight) if ctx.needs_input_grad[2] else None
        gb = torch.empty_like(bias) if ctx.needs_input_grad[3] else None
        if l.numel() == 0:
            return dl, du, gw if gw is None else gw.zero_(), gb if gb is None else gb.zero_(), None, None, None
        with _on(l.device):
            need = lib.linf_group_norm_bound_workspace_bytes(*sizes, 1)
            ws = _scratch(l.device, need)
            rc = lib.linf_group_norm_bound_backward(gl.data_ptr(), gu.data_ptr(), l.data_ptr(), u.data_ptr(), _ptr(weight), _ptr(bias),
                                                    sums.data_ptr(), *sizes, eps, act, _ptr(dl), _ptr(du), _ptr(gw), _ptr(gb), ws.data_ptr(),
                                                    need, _stream())
        _lib.check(rc, "group_norm_bound_backward")
        return (dl if ctx.needs_input_grad[0] else None, du if ctx.needs_input_grad[1] else None, gw, gb, None, None, None)


def _check_norm(x, name, groups, weight, bias, eps, activation):
    if x.dim() < 2:
        raise RuntimeError(f"{name} must be [N, C, ...]")
    groups, C = int(groups), x.size(1)
    if groups < 1 or C < 1 or C % groups != 0:
        raise ValueError("the channel count must be a multiple of the group count")
    if max(x.size(0), C, math.prod(x.shape[2:])) >= 2 ** 31:
        raise RuntimeError(f"each size of {name} must be below 2^31")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}")
    if not (math.isfinite(eps) and eps > 0):
        raise ValueError("eps must be finite and greater than 0")
    for v, what in ((weight, "weight"), (bias, "bias")):
        if v is None:
            continue
        if v.shape != (C,) or not v.is_contiguous():
            raise RuntimeError(f"{what} must be contiguous, with one element for each of the {C} channels")
        if v.device != x.device:
            raise RuntimeError(f"{what} must be on the device of {name}")
        if v.dtype not in (torch.float32, x.dtype):
            raise RuntimeError(f"{what} must have dtype torch.float32 or that of {name}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("weight and bias must have one dtype")
    _floating(x, name)
    return groups, float(eps), ACTIVATIONS[activation]


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation="identity", rate=0.0, rng=None):
    """activation((x - mean) / sqrt(var + eps) * weight + bias), mean and var over the positions and the C / groups neighbouring
    channels of a sample's group; x [N, C, ...] in fp32, fp16 or bf16, weight and bias [C] in fp32 or the type of x.

    activation: "identity", "relu", "tanh" or "silu".  rate > 0 drops elements of the result under rng {seed, offset} in the same pass:
    what `dropout(y, rate, rng)` gives.  Computed in fp32 and rounded once.  Channels-last memory is taken as it is, any
    other layout is copied to it; the result has its channels last in memory."""
    rate = _rate(rate)
    if rate > 0:
        if rng is None:
            raise RuntimeError("a rate above 0 needs rng, an int64 tensor of seed and offset")
        _generator_state(rng, x.device)
    groups, eps, act = _check_norm(x, "x", groups, weight, bias, eps, activation)
    return GroupNormF.apply(x, weight, bias, groups, eps, act, rate, rng if rate > 0 else None)


def group_norm_bound(lower, upper, groups, weight=None, bias=None, eps=1e-5, activation="identity"):
    """Bounds (lower, upper) of `group_norm` over every input between `lower` and `upper`, with gradients; fp32.

    The exact range of x_i - mean(x) over the box is divided by a range of the deviation that the triangle inequality gives, so the
    bounds hold for the box as a whole and collapse to the value where lower = upper; nothing normalised exceeds sqrt(M - 1) in a
    group of M.  Computed in 64 bits and rounded once, to nearest (as the bounds of the other layers are)."""
    if upper.shape != lower.shape or upper.dtype != lower.dtype or upper.device != lower.device:
        raise RuntimeError("upper must have the shape, dtype and device of lower")
    if lower.dtype != torch.float32:
        raise RuntimeError("bounds must have dtype torch.float32")
    groups, eps, act = _check_norm(lower, "lower", groups, weight, bias, eps, activation)
    return GroupNormBoundF.apply(lower, upper, weight, bias, groups, eps, act)


class BoundGroupNorm(_Masks):
    """Group norm with an activation on a triple (value, lower, upper); with `dropout` > 0 the triple is dropped under one mask
    while training.  state_dict: weight, bias [channels] if affine, rng where there is dropout."""

    def __init__(self, groups, channels, eps=1e-5, affine=True, activation="identity", dropout=0.0, seed=None):
        super().__init__()
        if groups < 1 or channels % groups != 0:
            raise ValueError("the channel count must be a multiple of the group count")
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}")
        self.groups, self.channels, self.eps, self.activation = groups, channels, eps, activation
        self.weight = nn.Parameter(torch.ones(channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(channels)) if affine else None
        self._make_masks(dropout, seed)

    def forward(self, x, lower=None, upper=None):
        args = (self.groups, self.weight, self.bias, self.eps, self.activation)
        rate = self.rate if self.training else 0.0
        used = dropout_next(self.rng) if rate > 0 else None
        if lower is None or upper is None:
            return group_norm(x, *args, rate, used), None, None
        lo, up = group_norm_bound(lower, upper, *args)
        if rate > 0:
            lo, up = DropoutF.apply(rate, used, lo, up)
        if skips_values() and not self.training and not torch.is_grad_enabled():
            return lo, lo, up                 # nobody reads the value in such a pass
        return group_norm(x, *args, rate, used), lo, up

    def extra_repr(self):
        s = f"{self.groups}, {self.channels}, eps={self.eps}, activation={self.activation}"
        return s + (f", dropout={self.rate}" if self.rate > 0 else "")
