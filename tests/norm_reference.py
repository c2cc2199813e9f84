"""Plain implementations in 64 bits, on the CPU, of the operators between two layers (group norm, its interval form, dropout),
and how far an implementation that computes in 32 bits may be from them.  Written from the formulas; gradients by autograd."""
import math

import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}     # half a step next to 0, or less
E = 2.0 ** -24
SILU_ARG = -1.278464542761074


def threshold(rate):
    return int(math.floor(rate * 65536 + 0.5))


def pieces(seed, offset, count, first=0):
    """The generator's 16-bit pieces of elements first .. first + count - 1 (first a multiple of 8): Philox4x32 with 7 rounds."""
    u = np.uint64
    low = u(0xFFFFFFFF)
    i = np.arange((count + 7) // 8, dtype=np.uint64) + u(first // 8)
    seed, offset = u(seed & (2 ** 64 - 1)), u(offset & (2 ** 64 - 1))
    c = [i & low, i >> u(32), np.full_like(i, offset & low), np.full_like(i, offset >> u(32))]
    k = [int(seed & low), int(seed >> u(32))]
    for _ in range(7):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(k[0]), b & low, (a >> u(32)) ^ c[3] ^ u(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack([p for w in c for p in (w & u(0xFFFF), w >> u(16))], axis=1).reshape(-1)[:count].astype(np.int64)


def kept(seed, offset, count, rate, first=0):
    return torch.from_numpy(pieces(seed, offset, count, first) >= threshold(rate))


def scale(rate):
    return 65536.0 / (65536.0 - threshold(rate)) if threshold(rate) < 65536 else 0.0


def rows(t):
    """[N, C, ...] -> [N, L, C]"""
    return t.reshape(t.size(0), t.size(1), -1).transpose(1, 2)


def unrows(t, shape):
    return t.transpose(1, 2).reshape(shape)


def activate(u, act):
    return {"identity": lambda t: t, "relu": torch.relu, "tanh": torch.tanh, "silu": torch.nn.functional.silu}[act](u)


def norm_parts(x, groups, weight, bias, eps):
    """(mean, 1 / deviation, h, u), each broadcast to [N, C, ...], in 64 bits."""
    N, C = x.shape[:2]
    t = x.reshape(N, groups, -1)
    mean = t.mean(dim=2, keepdim=True)
    r = 1.0 / (((t - mean) ** 2).mean(dim=2, keepdim=True) + eps).sqrt()
    h = ((t - mean) * r).reshape(x.shape)
    c = [1, C] + [1] * (x.dim() - 2)
    u = h * (weight.view(c) if weight is not None else 1.0) + (bias.view(c) if bias is not None else 0.0)
    wide = lambda s: s.expand(t.shape).reshape(x.shape)  # noqa: E731
    return wide(mean), wide(r), h, u


def group_norm(x, groups, weight, bias, eps, act, factor=None):
    y = activate(norm_parts(x, groups, weight, bias, eps)[3], act)
    return y if factor is None else y * factor


def bound_parts(lower, upper, groups, weight, bias, eps):
    """(v-, v+) in 64 bits."""
    shape, C = lower.shape, lower.size(1)
    l, u = lower.reshape(shape[0], groups, -1), upper.reshape(shape[0], groups, -1)
    M = l.size(2)
    c, r = (l + u) / 2, (u - l) / 2
    sd = ((c - c.mean(2, keepdim=True)) ** 2).mean(2, keepdim=True).clamp(min=1e-300).sqrt()
    rho = (r * r).mean(2, keepdim=True).clamp(min=1e-300).sqrt()
    wide, tight = ((sd + rho) ** 2 + eps) ** -0.5, ((sd - rho).clamp(min=0) ** 2 + eps) ** -0.5
    n0 = (l * (M - 1) - (u.sum(2, keepdim=True) - u)) / M
    n1 = (u * (M - 1) - (l.sum(2, keepdim=True) - l)) / M
    cut = math.sqrt(M - 1)
    z0 = torch.where(n0 >= 0, n0 * wide, n0 * tight)
    z1 = torch.where(n1 >= 0, n1 * tight, n1 * wide)
    z0 = torch.where(z0 <= -cut, torch.full_like(z0, -cut), z0).reshape(shape)
    z1 = torch.where(z1 >= cut, torch.full_like(z1, cut), z1).reshape(shape)
    k = [1, C] + [1] * (lower.dim() - 2)
    w = weight.view(k) if weight is not None else torch.ones(k, dtype=torch.float64)
    b = bias.view(k) if bias is not None else torch.zeros(k, dtype=torch.float64)
    v0, v1 = z0 * w + b, z1 * w + b
    turned = (w < 0).expand(shape)
    return torch.where(turned, v1, v0), torch.where(turned, v0, v1)


def group_norm_bound(lower, upper, groups, weight, bias, eps, act):
    v0, v1 = bound_parts(lower, upper, groups, weight, bias, eps)
    y0, y1 = activate(v0, act), activate(v1, act)
    if act == "silu":
        low = torch.where(y0 <= y1, y0, y1)
        low = torch.where((v0 < SILU_ARG) & (v1 > SILU_ARG), activate(torch.full_like(v0, SILU_ARG), act), low)
        return low, torch.where(y1 > y0, y1, y0)
    return y0, y1


# ---- how far 32-bit arithmetic may be off ---------------------------------------------------------------------------------


def error_of_u(mean, r, h, u, weight):
    """h = (x - mean) r: the mean rounded to fp32 (E |mean|) and the difference (E |x - mean|, r of it is |h|), the 64-bit sums' r
    rounded (E), the product (E); then the fused product with the weight and the sum (E |u|).  Squares of E are left out, twice the sum
    is allowed for them and for the order of the two products."""
    eh = 2 * E * (3 * h.abs() + r * mean.abs())
    c = [1, -1] + [1] * (h.dim() - 2)
    w = weight.abs().view(c) if weight is not None else 1.0
    return eh, w * eh + 2 * E * u.abs()


def error_of_act(u, eu, act):
    """No slope of the activations is above 1.1.  tanhf is off by at most 2 steps (4 E relative).  The sigmoid's exponential is off
    by 2 + 1.173 |u| steps (of 2 E), its sum by E, its division by 2 steps: times |silu(u)|."""
    y = activate(u, act).abs()
    own = {"identity": 0.0, "relu": 0.0, "tanh": 4 * E * y, "silu": 2 * E * (6 + 1.2 * u.abs()) * y}[act]
    return 1.1 * eu + own


def error_of_slope(u, eu, act):
    """No second derivative is above 1.  tanh: 1 - t^2 with t off by 4 E; silu: q (1 + u (1 - q)) with q off by 2 E (6 + 1.2 |u|) of
    itself, which moves the slope by at most (1 + 2 |u|) times that."""
    own = {"identity": 0.0, "relu": 0.0, "tanh": 16 * E, "silu": 2 * E * (8 + 1.2 * u.abs()) * (1 + 2 * u.abs())}[act]
    return (0.0 if act in ("identity", "relu") else eu) + own


def rounded(t, dtype):
    """Half a step of the result's type."""
    return HALF_STEP[dtype] * t.abs() + LEAST[dtype]
