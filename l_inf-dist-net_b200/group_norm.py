"""Group norm with an activation (and dropout) in the same pass, channels last, and its interval form.

Beside the mean shift (MeanNorm, BoundMeanNorm): where a net needs the spread of its activations normalised as well, per sample,
so that evaluation and training compute the same.  A group norm is not 1-Lipschitz in the sup norm as a distance layer is: its
place is the head behind the distance layers, and a certificate takes its bounds from `group_norm_bound`.
zbh2047/L_inf-dist-net has no counterpart.  Kernels: csrc/group_norm.cu, csrc/group_norm_bound.cu.
"""
import math
import operator

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _lib
from .dropout import DropoutTripleF, _Masks, _TYPES, _floating, _generator_state, _not_traced, _once, _rate, dropout_next
from .norm_dist import _on, _scratch, _stream, skips_values

ACTIVATIONS = {"identity": 0, "relu": 1, "tanh": 2, "silu": 3}        # LINF_ACT_*


def _rows(t):
    """[N, C, ...] -> the tensor itself where its channels lie last in memory, or a copy for which they do."""
    dims = t.dim()
    if t.is_contiguous() if dims == 2 else t.is_contiguous(memory_format=torch.channels_last) if dims == 4 else t.movedim(1, -1).is_contiguous():
        return t
    return t.movedim(1, -1).contiguous().movedim(-1, 1)


class _Call:
    """What a call has besides its tensors.  sizes: (N, C, groups, positions)."""
    __slots__ = ("sizes", "type", "param_type", "eps", "act", "rate", "rng")


_workspace_bytes = {}


def _work_space(query, device, *key):
    """Scratch of a call (from the current stream's pool), or None where it needs none; what a call needs is asked once."""
    need = _workspace_bytes.get((query, device.index, key))
    if need is None:
        if len(_workspace_bytes) >= 4096:
            _workspace_bytes.clear()
        need = _workspace_bytes[query, device.index, key] = getattr(_lib.load(), query)(*key)
    return _scratch(device, need) if need else None, need


def _ptr(t):
    return None if t is None else t.data_ptr()


def _norm_forward(call, x, weight, bias, keep):
    """The result, and with `keep` what the backward pass needs of it."""
    rows = _rows(x)
    y = torch.empty_like(rows)
    sizes = call.sizes
    stats = torch.empty(2, sizes[0], sizes[2], device=x.device, dtype=torch.float32) if keep else None
    if x.numel() > 0:
        with _on(x.device):
            ws, need = _work_space("linf_group_norm_workspace_bytes", x.device, *sizes, call.type, 0)
            at = stats.data_ptr() if keep else 0
            rc = _lib.load().linf_group_norm_forward(
                rows.data_ptr(), _ptr(weight), _ptr(bias), *sizes, call.type, call.param_type, call.eps, call.act, call.rate, _ptr(call.rng),
                y.data_ptr(), at or None, at + 4 * sizes[0] * sizes[2] if keep else None, _ptr(ws), need, _stream())
        _lib.check(rc, "group_norm_forward")
    return y, rows, stats


class GroupNormF(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, call):
        y, rows, stats = _norm_forward(call, x, weight, bias, True)
        ctx.call, ctx.stats = call, stats
        ctx.save_for_backward(rows, weight, bias, call.rng)
        return y

    @staticmethod
    @_once
    def backward(ctx, grad_output):
        call = ctx.call
        rows, weight, bias, rng = ctx.saved_tensors
        sizes = call.sizes
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        g = _rows(grad_output)
        gx = torch.empty_like(rows) if need_x else None
        gw = torch.empty_like(weight) if need_w else None
        gb = torch.empty_like(bias) if need_b else None
        if rows.numel() == 0:
            return gx, gw if gw is None else gw.zero_(), gb if gb is None else gb.zero_(), None
        with _on(rows.device):
            ws, need = _work_space("linf_group_norm_workspace_bytes", rows.device, *sizes, call.type, 1)
            at = ctx.stats.data_ptr()
            rc = _lib.load().linf_group_norm_backward(
                g.data_ptr(), rows.data_ptr(), _ptr(weight), _ptr(bias), at, at + 4 * sizes[0] * sizes[2], *sizes, call.type, call.param_type,
                call.act, call.rate, _ptr(rng), _ptr(gx), _ptr(gw), _ptr(gb), _ptr(ws), need, _stream())
        _lib.check(rc, "group_norm_backward")
        return gx, gw, gb, None


def _bound_forward(call, lower, upper, weight, bias, keep):
    l, u = _rows(lower), _rows(upper)
    lo, up = torch.empty_like(l), torch.empty_like(l)
    sizes = call.sizes
    sums = torch.empty(sizes[0], sizes[2], 4, device=l.device, dtype=torch.float64) if keep else None
    if l.numel() > 0:
        with _on(l.device):
            ws, need = _work_space("linf_group_norm_bound_workspace_bytes", l.device, *sizes, 0)
            rc = _lib.load().linf_group_norm_bound_forward(l.data_ptr(), u.data_ptr(), _ptr(weight), _ptr(bias), *sizes, call.eps, call.act,
                                                           lo.data_ptr(), up.data_ptr(), _ptr(sums), _ptr(ws), need, _stream())
        _lib.check(rc, "group_norm_bound_forward")
    return lo, up, l, u, sums


class GroupNormBoundF(torch.autograd.Function):

    @staticmethod
    def forward(ctx, lower, upper, weight, bias, call):
        lo, up, l, u, sums = _bound_forward(call, lower, upper, weight, bias, True)
        ctx.call, ctx.sums = call, sums
        ctx.save_for_backward(l, u, weight, bias)
        return lo, up

    @staticmethod
    @_once
    def backward(ctx, grad_lower, grad_upper):
        call = ctx.call
        l, u, weight, bias = ctx.saved_tensors
        sizes = call.sizes
        need_l, need_u, need_w, need_b, _ = ctx.needs_input_grad
        gl, gu = _rows(grad_lower), _rows(grad_upper)
        dl, du = (torch.empty_like(l), torch.empty_like(l)) if need_l or need_u else (None, None)
        gw = torch.empty_like(weight) if need_w else None
        gb = torch.empty_like(bias) if need_b else None
        if l.numel() == 0:
            return dl, du, gw if gw is None else gw.zero_(), gb if gb is None else gb.zero_(), None
        with _on(l.device):
            ws, need = _work_space("linf_group_norm_bound_workspace_bytes", l.device, *sizes, 1)
            rc = _lib.load().linf_group_norm_bound_backward(gl.data_ptr(), gu.data_ptr(), l.data_ptr(), u.data_ptr(), _ptr(weight), _ptr(bias),
                                                            ctx.sums.data_ptr(), *sizes, call.eps, call.act, _ptr(dl), _ptr(du), _ptr(gw), _ptr(gb),
                                                            _ptr(ws), need, _stream())
        _lib.check(rc, "group_norm_bound_backward")
        return dl if need_l else None, du if need_u else None, gw, gb, None


_checked = {}


def _check_sizes(shape, name, groups, eps, activation):
    """(sizes, activation's number, eps) of a call; what was found once for a shape is kept."""
    groups, eps = operator.index(groups), float(eps)
    key = (shape, groups, eps, activation)
    found = _checked.get(key)
    if found is not None:
        return found
    if len(shape) < 2:
        raise RuntimeError(f"{name} must be [N, C, ...]")
    C, positions = shape[1], math.prod(shape[2:])
    if groups < 1 or C < 1 or C % groups != 0:
        raise ValueError("the channel count must be a multiple of the group count")
    if max(shape[0], positions) > 2 ** 30 or C >= 2 ** 31:
        raise RuntimeError(f"{name} may have 2^30 samples, 2^30 positions and 2^31 - 1 channels at most")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}")
    if not 1.1754943508222875e-38 <= eps <= 3.4028234663852886e38:
        raise ValueError("eps must be a positive normal fp32 number")
    if len(_checked) >= 4096:
        _checked.clear()
    found = _checked[key] = ((shape[0], C, groups, positions), ACTIVATIONS[activation], eps)
    return found


def _make_call(x, name, groups, weight, bias, eps, activation):
    """Checks the arguments; what the kernels are to be told of them."""
    call = _Call()
    call.sizes, call.act, call.eps = _check_sizes(x.shape, name, groups, eps, activation)
    call.rate, call.rng, call.param_type = 0.0, None, 0
    C, dtype, device = call.sizes[1], x.dtype, x.device
    for v, what in ((weight, "weight"), (bias, "bias")):
        if v is None:
            continue
        if v.dim() != 1 or v.size(0) != C or not v.is_contiguous():
            raise RuntimeError(f"{what} must be contiguous, with one element for each of the {C} channels")
        if v.device != device:
            raise RuntimeError(f"{what} must be on the device of {name}")
        if v.dtype != torch.float32:
            if v.dtype != dtype:
                raise RuntimeError(f"{what} must have dtype torch.float32 or that of {name}")
            call.param_type = _TYPES.get(dtype, 0)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("weight and bias must have one dtype")
    _floating(x, name)
    call.type = _TYPES[dtype]
    return call


def _wants_grad(*tensors):
    """Whether the call has to go through its autograd function: for a backward pass, or because a tensor carries a forward-mode
    tangent (which the function refuses; the launch alone would lose it)."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation="identity", rate=0.0, rng=None):
    """activation((x - mean) / sqrt(var + eps) * weight + bias), mean and var over the positions and the C / groups neighbouring
    channels of a sample's group; x [N, C, ...] in fp32, fp16 or bf16, weight and bias [C] in fp32 or the type of x.

    activation: "identity", "relu", "tanh" or "silu".  rate > 0 drops elements of the result under rng {seed, offset} in the same pass:
    what `dropout(y, rate, rng)` gives.  Computed in fp32 and rounded once.  Channels-last memory is taken as it is, any
    other layout is copied to it; the result has its channels last in memory."""
    _not_traced("group_norm")
    rate = _rate(rate)
    if rate > 0:
        if rng is None:
            raise RuntimeError("a rate above 0 needs rng, an int64 tensor of seed and offset")
        _generator_state(rng, x.device)
    call = _make_call(x, "x", groups, weight, bias, eps, activation)
    if rate > 0:
        call.rate, call.rng = rate, rng
    if _wants_grad(x, weight, bias):
        return GroupNormF.apply(x, weight, bias, call)
    return _norm_forward(call, x, weight, bias, False)[0]


def group_norm_bound(lower, upper, groups, weight=None, bias=None, eps=1e-5, activation="identity"):
    """Bounds (lower, upper) of `group_norm` over every input between `lower` and `upper`, with gradients; fp32.

    The exact range of x_i - mean(x) over the box is divided by a range of the deviation that the triangle inequality gives, so the
    bounds hold for the box as a whole and collapse to the value where lower = upper; nothing normalised exceeds sqrt(M - 1) in a
    group of M.  The sums are 64-bit, the bounds fp32, rounded to nearest (as the bounds of the other layers are)."""
    _not_traced("group_norm_bound")
    if upper.shape != lower.shape or upper.dtype != lower.dtype or upper.device != lower.device:
        raise RuntimeError("upper must have the shape, dtype and device of lower")
    if lower.dtype != torch.float32:
        raise RuntimeError("bounds must have dtype torch.float32")
    call = _make_call(lower, "lower", groups, weight, bias, eps, activation)
    if _wants_grad(lower, upper, weight, bias):
        return GroupNormBoundF.apply(lower, upper, weight, bias, call)
    return _bound_forward(call, lower, upper, weight, bias, False)[:2]


class BoundGroupNorm(_Masks):
    """Group norm with an activation on a triple (value, lower, upper); with `dropout` > 0 the triple is dropped under one mask
    while training.  state_dict: weight, bias [channels] if affine, rng where there is dropout."""

    def __init__(self, groups, channels, eps=1e-5, affine=True, activation="identity", dropout=0.0, seed=None):
        super().__init__()
        groups = operator.index(groups)
        if groups < 1 or channels % groups != 0:
            raise ValueError("the channel count must be a multiple of the group count")
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}")
        self.groups, self.channels, self.eps, self.activation = groups, channels, eps, activation
        self.weight = nn.Parameter(torch.ones(channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(channels)) if affine else None
        self._make_masks(dropout, seed)

    def forward(self, x, lower=None, upper=None):
        if x.size(1) != self.channels:
            raise RuntimeError(f"the input must have {self.channels} channels")
        args = (self.groups, self.weight, self.bias, self.eps, self.activation)
        rate = self.rate if self.training else 0.0
        used = dropout_next(self.rng, self.replica) if rate > 0 else None
        if lower is None or upper is None:
            return group_norm(x, *args, rate, used), None, None
        lo, up = group_norm_bound(lower, upper, *args)
        if rate > 0:
            lo, up, _ = DropoutTripleF.apply(rate, used, lo, up, None)
        if skips_values() and not self.training and not torch.is_grad_enabled():
            return lo, lo, up                 # nobody reads the value in such a pass
        return group_norm(x, *args, rate, used), lo, up

    def extra_repr(self):
        s = f"{self.groups}, {self.channels}, eps={self.eps}, activation={self.activation}"
        return s + (f", dropout={self.rate}" if self.rate > 0 else "")
