"""Dropout whose mask is a function of (seed, offset, element number) and is never stored: forward and backward compute it
again (csrc/dropout.cu; the generator is Philox4x32 with 7 rounds, 16 bits for each element).

Beside the elementwise maps of the heads (BoundReLU, BoundTanh): `BoundDropout` maps a triple (value, lower, upper) under ONE
mask, so that lower <= value <= upper still holds behind it.  zbh2047/L_inf-dist-net has no counterpart.
"""
import threading

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib
from .norm_dist import _on, _stream

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}      # LINF_F32, LINF_F16, LINF_BF16


def _once(backward):
    """A backward pass that may be differentiated no further (once_differentiable, without its guard where no graph is made of it)."""
    checked = once_differentiable(backward)

    def run(ctx, *grads):
        return checked(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def _not_traced(name):
    """torch.jit.trace sees the allocation of a result and not the launch that fills it."""
    if torch.jit.is_tracing():
        raise RuntimeError(f"{name} cannot be traced by torch.jit")


def _floating(t, name):
    if t.dtype not in _TYPES:
        raise RuntimeError(f"{name} must have dtype torch.float32, torch.float16 or torch.bfloat16")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")


def _generator_state(rng, device):
    if not (torch.is_tensor(rng) and rng.dtype == torch.int64 and rng.shape == (2,) and rng.is_contiguous()):
        raise RuntimeError("rng must be a contiguous int64 tensor of two elements: seed and offset")
    if rng.device != device:
        raise RuntimeError("rng must be on the device of the tensors it drops elements of")


def _rate(rate):
    rate = float(rate)
    if not 0.0 <= rate <= 1.0:
        raise ValueError("the dropout rate must lie in [0, 1]")
    return rate


def _is_last(t):
    """Whether the channels (dimension 1) lie last in memory, without gaps."""
    return t.dim() > 2 and t.movedim(1, -1).is_contiguous()


def _as_stored(t, last):
    """t with its elements in memory order: as it is, or a copy."""
    if t.is_contiguous() if not last else _is_last(t):
        return t
    return t.contiguous() if not last else t.movedim(1, -1).contiguous().movedim(-1, 1)


def _launch(rate, rng, a, b=None, c=None):
    """The mask on up to three tensors (each may be None); as many results."""
    some = a if a is not None else b if b is not None else c
    if some is None:
        return None, None, None
    outs = [None if t is None else torch.empty_like(t) for t in (a, b, c)]
    if some.numel() > 0:
        ptr = [None if t is None else t.data_ptr() for t in (a, b, c, *outs)]
        with _on(some.device):
            rc = _lib.load().linf_dropout(*ptr[:3], some.numel(), _TYPES[some.dtype], rate, rng.data_ptr(), *ptr[3:], _stream())
        _lib.check(rc, "dropout")
    return outs


class DropoutF(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, rate, rng):
        last = not x.is_contiguous() and _is_last(x)
        ctx.last, ctx.rate = last, rate
        ctx.save_for_backward(rng)
        return _launch(rate, rng, _as_stored(x, last))[0]

    @staticmethod
    @_once
    def backward(ctx, grad):
        rng, = ctx.saved_tensors
        return _launch(ctx.rate, rng, _as_stored(grad, ctx.last))[0], None, None


class DropoutTripleF(torch.autograd.Function):
    """The same mask on up to three tensors (c may be None)."""

    @staticmethod
    def forward(ctx, rate, rng, a, b, c):
        ctx.set_materialize_grads(False)
        last = not a.is_contiguous() and _is_last(a)
        ctx.last, ctx.rate = last, rate
        ctx.save_for_backward(rng)
        return tuple(_launch(rate, rng, *[None if t is None else _as_stored(t, last) for t in (a, b, c)]))

    @staticmethod
    @_once
    def backward(ctx, *grads):
        rng, = ctx.saved_tensors
        given = [_as_stored(g, ctx.last) if need and g is not None else None for g, need in zip(grads, ctx.needs_input_grad[2:])]
        return (None, None, *_launch(ctx.rate, rng, *given))


_masks_of = threading.local()          # .stack: the blocks of `checkpoint_masks` that this thread is in, the innermost last


class _Drawn:
    """A block of `checkpoint_masks`: where the pairs that are drawn in it are kept, or, `again`, from where they come once more."""

    def __init__(self, pairs, again):
        self.pairs, self.again, self.at = pairs, again, 0

    def __enter__(self):
        self.at = 0
        if not hasattr(_masks_of, "stack"):
            _masks_of.stack = []
        _masks_of.stack.append(self)
        return self

    def __exit__(self, *exc):
        _masks_of.stack.pop()

    def take(self, state):
        if self.at == len(self.pairs) or self.pairs[self.at][0] is not state:
            raise RuntimeError("the checkpointed function draws other masks when it is run again than it did at first")
        self.at += 1
        return self.pairs[self.at - 1][1]


def checkpoint_masks():
    """The `context_fn` with which `torch.utils.checkpoint.checkpoint(..., use_reentrant=False)` runs a function that drops elements: the second run
    gets the pairs of the first, and with them its masks.  Without it a pass that is run again is refused, for it would draw others."""
    pairs = []
    return _Drawn(pairs, False), _Drawn(pairs, True)


def _draw(state, replica):
    if not state.is_cuda:
        raise RuntimeError("rng must be a CUDA tensor")
    used = torch.empty_like(state)
    with _on(state.device):
        rc = _lib.load().linf_dropout_next_replica(state.data_ptr(), replica, used.data_ptr(), _stream())
    _lib.check(rc, "dropout_next")
    torch.autograd.graph.increment_version(state)       # a backward pass that was to read `state` itself is refused by autograd
    return used


def dropout_next(state, replica=0):
    """{seed, offset} to draw one mask with, as a tensor of its own; the offset of `state` rises by 1.  Runs on the device, so a
    captured graph draws another mask each time it is replayed, and calls on several streams never get the same offset.
    replica: its number among those that hold equal states, each of which gets a seed of its own.

    Within a backward pass (a checkpointed function that is run again) it is refused, or gives what it gave at first: `checkpoint_masks`."""
    _not_traced("dropout_next")
    _generator_state(state, state.device)
    used, keep = None, []
    for block in reversed(getattr(_masks_of, "stack", ())):
        if block.again:
            used = block.take(state)
            break
        keep.append(block)
    if used is None:
        if torch._C._current_graph_task_id() != -1:
            raise RuntimeError("a mask is drawn within a backward pass: a checkpointed function that drops elements needs use_reentrant=False and "
                               "context_fn=checkpoint_masks")
        used = _draw(state, replica)
    for block in keep:
        block.pairs.append((state, used))
    return used


def dropout(x, rate, rng, lower=None, upper=None):
    """x with each element dropped (0) with probability `rate`, the others multiplied by 1 / (1 - rate); with lower / upper the
    triple under one mask.  fp32, fp16 or bf16.

    rng: int64 CUDA tensor {seed, offset}; the same pair gives the same mask (see `dropout_next`), and it has to hold its values
    until the backward pass.  Rates count in steps of 2^-16, the scale makes up for that.  Elements are numbered as they lie
    in memory where x is contiguous or has its channels last; another layout is copied to a contiguous one first, and
    lower / upper to the layout of x."""
    rate = _rate(rate)
    if (lower is None) != (upper is None):
        raise RuntimeError("lower and upper are given together")
    if lower is not None:
        for t, name in ((lower, "lower"), (upper, "upper")):
            if t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
                raise RuntimeError(f"{name} must have the shape, dtype and device of x")
    _generator_state(rng, x.device)
    _floating(x, "x")
    if lower is None:
        return DropoutF.apply(x, rate, rng)
    return DropoutTripleF.apply(rate, rng, x, lower, upper)


class _Masks(nn.Module):
    """Keeps the generator state of a module that drops elements: a buffer `rng` of {seed, offset}.  `replica`: the module's number among
    the replicas of a data-parallel job (the step classes of train_step.py set it; with another wrapper, the program does).  It is no part of the
    state, which the ranks load, or broadcast to each other, as it is."""

    replica = 0

    def _make_masks(self, rate, seed):
        self.rate = _rate(rate)
        if self.rate > 0:
            seed = int(torch.randint(0, 2 ** 62, ())) if seed is None else int(seed)
            self.register_buffer("rng", torch.tensor([seed, 0], dtype=torch.int64))


class BoundDropout(_Masks):
    """Dropout of a triple (value, lower, upper) while training; nothing in eval mode.  Every forward pass draws a mask of its own.
    seed: by default a number from torch's CPU generator.  Replicas of a data-parallel job may have equal ones (`replica`)."""

    def __init__(self, rate, seed=None):
        super().__init__()
        self._make_masks(rate, seed)

    def forward(self, x, lower=None, upper=None):
        if lower is None or upper is None:
            lower = upper = None
        if not self.training or self.rate == 0:
            return x, lower, upper
        used = dropout_next(self.rng, self.replica)
        if lower is None:
            return dropout(x, self.rate, used), None, None
        return dropout(x, self.rate, used, lower, upper)

    def extra_repr(self):
        return f"rate={self.rate}"
