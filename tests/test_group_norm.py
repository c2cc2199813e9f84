"""Group norm with an activation and dropout, and its interval form, against plain implementations in 64 bits; refusals; layouts,
streams, graphs; the head and the convolution that use them.  The tolerances are worked out in norm_reference.py and below."""
import ctypes
import math

import pytest
import torch

import linfdist_b200 as L
import norm_reference as R
from norm_reference import E

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
EPS = 1e-5

# (N, C, groups, positions): one value in a group; one channel in a group; groups no vector divides; groups over several vectors;
# odd channel counts; groups of more vectors than a CTA has threads; one position; many positions; many samples
SHAPES = [(1, 1, 1, (1,)), (2, 4, 4, ()), (3, 6, 3, ()), (5, 30, 3, (5, 7)), (2, 64, 8, (16, 16)), (3, 75, 5, (37,)), (2, 40, 4, (9, 9)),
          (2, 320, 32, (8, 8)), (1, 2048, 2048, (3,)), (7, 512, 16, ()), (3, 5120, 1, ()), (2, 8200, 1, (2,)), (2, 2666, 2, (3,)),
          (1, 6144, 2, (5,)), (1, 16, 2, (150, 150)), (1, 3, 1, (101, 103)), (3000, 8, 2, ()),
          # rows too wide for a CTA's threads; small samples of which a CTA takes several; parts of the rows of several samples; one channel
          (2, 20000, 1, ()), (5000, 32, 4, (3,)), (3, 48, 6, (60, 61)), (2, 1, 1, (200, 90)),
          # vectors of 8 and 4 bytes
          (2, 36, 3, (9, 5)), (1, 20, 2, (70, 90)), (6, 44, 2, ()), (1, 18, 1, (80, 90)), (2, 22, 11, (7,))]


def ids(s):
    return "N{}_C{}_G{}_{}".format(*s[:3], "x".join(map(str, s[3])) or "dense")


def make(shape, dtype, seed, spread=0.5, level=3.0):
    """Activations as distance layers give them (all positive), parameters, an output gradient; on the CPU."""
    N, C, groups, space = shape
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x = (level + 0.5 * rand(C).view(1, C, *[1] * len(space)) + spread * rand(N, C, *space)).to(dtype)
    return x, 1 + 0.3 * rand(C), 0.3 * rand(C), rand(N, C, *space).to(dtype)


def last(t):
    """The same tensor on the GPU with the channels last in memory."""
    return t.cuda().movedim(1, -1).contiguous().movedim(-1, 1)


def numbered(shape, seed, offset, rate):
    """Kept (1 / (1 - rate)) or dropped (0): elements are numbered with the channels last."""
    N, C = shape[:2]
    L_ = math.prod(shape[2:])
    keep = R.kept(seed, offset, N * C * L_, rate).view(N, L_, C)
    return R.unrows(keep.double() * R.scale(rate), shape)


def assert_within(got, want, most, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= most)
    if bad.any():
        k = ((got - want).abs() / most.clamp(min=1e-300)).argmax()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off; worst {got.reshape(-1)[k]:.9g} for "
                             f"{want.reshape(-1)[k]:.9g}, allowed {most.expand_as(want).reshape(-1)[k]:.3g}")


def reference(x, w, b, groups, act, g, factor=None):
    """Value, gradients, and what each may be off by."""
    xd = x.double().requires_grad_()
    wd, bd = (None if t is None else t.double().requires_grad_() for t in (w, b))
    y = R.group_norm(xd, groups, wd, bd, EPS, act, factor)
    leaves = [t for t in (xd, wd, bd) if t is not None]
    grads = torch.autograd.grad(y, leaves, g.double())
    with torch.no_grad():
        mean, r, h, u = R.norm_parts(xd, groups, wd, bd, EPS)
        eh, eu = R.error_of_u(mean, r, h, u, wd)
        f = torch.ones_like(y) if factor is None else factor
        most = [f * R.error_of_act(u, eu, act) + 2 * E * y.abs() + R.rounded(y, x.dtype)]
        # gradients: du = g f act'(u); a sum of n terms in 32 bits, partly in a tree, is off by at most 128 E of the terms' sizes
        # (a thread adds at most 64 values one after the other before 64-bit sums take over)
        with torch.enable_grad():
            ud = u.clone().requires_grad_()
            slope, = torch.autograd.grad(R.activate(ud, act).sum(), ud)
        du = g.double() * f * slope
        edu = (g.double() * f).abs() * R.error_of_slope(u, eu, act) + 3 * E * du.abs()
        c = [1, -1] + [1] * (x.dim() - 2)
        wa = 1.0 if wd is None else wd.abs().view(c)
        N = x.size(0)
        mean_of = lambda t: t.expand_as(h).reshape(N, groups, -1).mean(2, keepdim=True).expand(N, groups, h[0].numel() // groups).reshape(h.shape)  # noqa: E731
        q, eq = wa * du.abs(), wa * edu
        s1, s2 = mean_of(q), mean_of(q * h.abs())
        e1, e2 = mean_of(eq) + 130 * E * s1, mean_of(eq * h.abs() + q * eh) + 130 * E * s2
        gx = r * (eq + e1 + h.abs() * e2 + eh * s2 + 6 * E * (q + s1 + h.abs() * s2))
        most.append(gx + R.rounded(grads[0], x.dtype))
        over = [k for k in range(x.dim()) if k != 1]
        if w is not None:
            most.append((edu * h.abs() + du.abs() * eh + 130 * E * (du * h).abs()).sum(over) + R.rounded(grads[1], w.dtype))
        if b is not None:
            most.append((edu + 130 * E * du.abs()).sum(over) + R.rounded(grads[-1], b.dtype))
    return [y.detach(), *grads], most


def check(shape, dtype, act, seed, rate=0.0, give=last, params=True, ptype=torch.float32, spread=0.5, level=3.0):
    x, w, b, g = make(shape, dtype, seed, spread, level)
    w, b = (w.to(ptype), b.to(ptype)) if params else (None, None)
    factor = numbered(x.shape, 1000 + seed, 3, rate) if rate > 0 else None
    want, most = reference(x, w, b, shape[2], act, g, factor)
    leaves = [give(x).requires_grad_()] + [t.cuda().requires_grad_() for t in (w, b) if t is not None]
    rng = torch.tensor([1000 + seed, 3], dtype=torch.int64, device="cuda") if rate > 0 else None
    y = L.group_norm(leaves[0], shape[2], *(leaves[1:] if params else (None, None)), eps=EPS, activation=act, rate=rate, rng=rng)
    assert y.dtype == dtype and y.movedim(1, -1).is_contiguous()
    got = [y, *torch.autograd.grad(y, leaves, give(g))]
    for a, e, m, what in zip(got, want, most, ("value", "grad_x", "grad_weight", "grad_bias")):
        assert_within(a, e, m, f"{what} of {shape} {dtype} {act}")
    return got


# ---- on the host ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("act", ["identity", "tanh", "silu"])
def test_reference_gradients_against_differences(act):
    """The plain implementations' gradients are the slopes of their values."""
    gen = torch.Generator().manual_seed(1)
    x = (3 + torch.randn(2, 6, 5, generator=gen, dtype=torch.float64)).requires_grad_()
    w, b = (torch.randn(6, generator=gen, dtype=torch.float64).requires_grad_() for _ in range(2))
    torch.autograd.gradcheck(lambda *t: R.group_norm(t[0], 3, t[1], t[2], EPS, act), (x, w, b), eps=1e-6, atol=1e-6)
    lo, up = (x - 0.1).detach().requires_grad_(), (x + 0.2).detach().requires_grad_()
    torch.autograd.gradcheck(lambda *t: R.group_norm_bound(t[0], t[1], 3, t[2], t[3], EPS, act), (lo, up, w, b), eps=1e-6, atol=1e-6)


@pytest.mark.parametrize("act", ["identity", "relu", "tanh", "silu"])
def test_reference_bounds_hold(act):
    """Points of the box, its corners among them, stay within the bounds; a box of one point has the value as both bounds."""
    gen = torch.Generator().manual_seed(2)
    for groups, radius in ((1, 0.02), (2, 0.3), (4, 2.0), (8, 0.1)):
        lo = torch.randn(3, 8, 4, generator=gen, dtype=torch.float64)
        up = lo + radius * torch.rand(3, 8, 4, generator=gen, dtype=torch.float64)
        w, b = torch.randn(8, generator=gen, dtype=torch.float64), torch.randn(8, generator=gen, dtype=torch.float64)
        y0, y1 = R.group_norm_bound(lo, up, groups, w, b, EPS, act)
        for k in range(60):
            t = torch.rand(3, 8, 4, generator=gen, dtype=torch.float64)
            y = R.group_norm(lo + (up - lo) * (t.round() if k % 2 else t), groups, w, b, EPS, act)
            assert (y >= y0 - 1e-12).all() and (y <= y1 + 1e-12).all()
        y = R.group_norm(lo, groups, w, b, EPS, act)
        for end in R.group_norm_bound(lo, lo, groups, w, b, EPS, act):
            assert (end - y).abs().max() < 1e-9


def _refused(fn, base, cases):
    for change, code in cases:
        a = dict(base)
        a.update(change)
        assert fn(*a.values()) == code, change


def test_library_refuses(lib):
    p = ctypes.c_void_p(4096)          # never followed: each call is refused before a launch
    inf, nan = float("inf"), float("nan")
    sizes = [(dict(N=0), 2), (dict(C=-4), 2), (dict(G=0), 2), (dict(L=0), 2), (dict(G=3), 3), (dict(L=(1 << 30) + 1), 7), (dict(N=(1 << 30) + 1), 7)]
    common = sizes + [(dict(act=4), 11), (dict(act=-1), 11), (dict(L=1 << 20, ws=None), 6), (dict(L=1 << 20, ws=ctypes.c_void_p(4097)), 6), (dict(L=1 << 20, ws_bytes=8), 6)]
    eps = [(dict(eps=0.0), 10), (dict(eps=-1.0), 10), (dict(eps=1e-40), 10), (dict(eps=inf), 10), (dict(eps=nan), 10)]
    kinds = [(dict(type=3), 8), (dict(type=-1), 8), (dict(ptype=2), 8), (dict(rate=-1.0), 9), (dict(rate=nan), 9), (dict(rate=0.5), 9), (dict(rate=2.0), 9)]
    fwd = dict(x=p, w=p, b=p, N=2, C=8, G=2, L=4, type=0, ptype=0, eps=1e-5, act=0, rate=0.0, rng=None, y=p, mean=p, rstd=p, ws=p, ws_bytes=1 << 20, st=None)
    _refused(lib.linf_group_norm_forward, fwd, common + eps + kinds + [(dict(x=None), 1), (dict(y=None), 1), (dict(mean=None), 1)])
    back = dict(dy=p, x=p, w=p, b=p, mean=p, rstd=p, N=2, C=8, G=2, L=4, type=0, ptype=0, act=0, rate=0.0, rng=None, dx=p, dw=p, db=p, ws=p,
                ws_bytes=1 << 20, st=None)
    _refused(lib.linf_group_norm_backward, back, common + kinds + [(dict(dy=None), 1), (dict(rstd=None), 1), (dict(dx=None, dw=None, db=None), 1)])
    bound = dict(l=p, u=p, w=p, b=p, N=2, C=8, G=2, L=4, eps=1e-5, act=0, ol=p, ou=p, sums=p, ws=p, ws_bytes=1 << 20, st=None)
    _refused(lib.linf_group_norm_bound_forward, bound, common + eps + [(dict(u=None), 1), (dict(ol=None), 1)])
    bback = dict(gl=p, gu=p, l=p, u=p, w=p, b=p, sums=p, N=2, C=8, G=2, L=4, eps=1e-5, act=0, dl=p, du=p, dw=p, db=p, ws=p, ws_bytes=1 << 20, st=None)
    _refused(lib.linf_group_norm_bound_backward, bback, common + eps + [(dict(sums=None), 1), (dict(du=None), 1), (dict(dl=None, du=None, dw=None, db=None), 1)])
    assert lib.linf_group_norm_workspace_bytes(2, 8, 3, 4, 0, 0) == 0 and lib.linf_group_norm_workspace_bytes(2, 8, 2, 4, 9, 0) == 0


def test_python_refuses_on_the_host():
    x, w = torch.randn(2, 8, 3), torch.ones(8)
    for kw in (dict(groups=3), dict(groups=0), dict(groups=2, eps=0.0), dict(groups=2, eps=float("nan")), dict(groups=2, activation="gelu"),
               dict(groups=2, rate=1.5), dict(groups=2, rate=-0.1)):
        with pytest.raises(ValueError):
            L.group_norm(x, **kw)
    for kw in (dict(weight=torch.ones(7)), dict(weight=torch.ones(16)[::2]), dict(weight=w.double()), dict(weight=w, bias=w.half()), dict(rate=0.5),
               dict(rate=0.5, rng=torch.zeros(2)), dict(weight=w.half())):
        with pytest.raises(RuntimeError, match="weight|bias|rng"):
            L.group_norm(x, 2, **kw)
    with pytest.raises(TypeError):
        L.group_norm(torch.zeros(2, 5), 2.5)
    with pytest.raises(TypeError):
        L.BoundGroupNorm(2.5, 5)
    with pytest.raises(RuntimeError, match="N, C"):
        L.group_norm(torch.zeros(4), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        L.group_norm(x, 2, w, w)
    with pytest.raises(RuntimeError, match="dtype"):
        L.group_norm(x.double(), 2)
    with pytest.raises(RuntimeError, match="float32"):
        L.group_norm_bound(x.half(), x.half(), 2)
    with pytest.raises(RuntimeError, match="upper"):
        L.group_norm_bound(x, x[:1], 2)
    for bad in (dict(groups=3, channels=8), dict(groups=2, channels=8, activation="gelu"), dict(groups=2, channels=8, dropout=2.0)):
        with pytest.raises(ValueError):
            L.BoundGroupNorm(**bad)
    for rate in (-0.1, float("nan"), 1.5):
        for groups in (None, 2):
            with pytest.raises(ValueError):
                L.Predictor(6, 8, 3, groups=groups, dropout=rate)
    with pytest.raises(RuntimeError, match="16 channels"):
        L.BoundGroupNorm(2, 16, affine=False)(x)


def test_modules_state_on_the_host():
    assert set(L.BoundGroupNorm(2, 8).state_dict()) == {"weight", "bias"}
    assert set(L.BoundGroupNorm(2, 8, affine=False, dropout=0.1).state_dict()) == {"rng"}
    assert set(L.Predictor(6, 8, 3).state_dict()) == {"fc1.weight", "fc1.bias", "fc2.weight", "fc2.bias"}      # as ever
    assert {"norm.weight", "norm.bias"} <= set(L.Predictor(6, 8, 3, groups=2).state_dict())


# ---- on the GPU -----------------------------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=ids)
def test_values_and_gradients(cuda, lib, shape, dtype):
    check(shape, dtype, "silu", seed=sum(shape[:3]))


@gpu
@pytest.mark.parametrize("act", ["identity", "tanh"])
@pytest.mark.parametrize("shape", [SHAPES[3], SHAPES[5], SHAPES[9]], ids=ids)
def test_activations(cuda, lib, shape, act):
    check(shape, torch.float32, act, seed=7)
    check(shape, torch.bfloat16, act, seed=7)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_relu(cuda, lib, dtype):
    """The slope jumps at u = 0: seven values of distance 0.4 and more from there (weights 1, bias 0: u is h)."""
    x = torch.tensor([1.0, 2.0, 3.0, 5.0, 6.0, 7.0, 8.0, 1.0], dtype=dtype).view(1, 8)[:, torch.tensor([0, 5, 2, 6, 3, 1, 4, 7])]
    x = x.expand(3, 8).contiguous()
    g = torch.arange(24, dtype=torch.float32).view(3, 8).to(dtype) / 8
    want, most = reference(x, None, None, 1, "relu", g)
    xd = x.cuda().requires_grad_()
    y = L.group_norm(xd, 1, eps=EPS, activation="relu")
    assert_within(y, want[0], most[0], "value")
    assert_within(torch.autograd.grad(y, xd, g.cuda())[0], want[1], most[1], "grad_x")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [SHAPES[1], SHAPES[3], SHAPES[4], SHAPES[5], SHAPES[7], SHAPES[9], SHAPES[12]], ids=ids)
def test_with_dropout(cuda, lib, shape, dtype):
    got = check(shape, dtype, "silu", seed=5, rate=0.3)
    # the same as dropout behind it, mask and all
    x, w, b, _ = make(shape, dtype, 5)
    rng = torch.tensor([1005, 3], dtype=torch.int64, device="cuda")
    two = L.dropout(L.group_norm(last(x), shape[2], w.cuda(), b.cuda(), EPS, "silu"), 0.3, rng)
    assert torch.equal(got[0] == 0, two == 0)
    if dtype == torch.float32:
        assert torch.equal(got[0], two)


@gpu
def test_layouts(cuda, lib):
    """Plain NCHW memory, slices, a tensor off a 16-byte boundary, a gradient in another layout."""
    shape = (3, 24, 4, (6, 5))
    plain = check(shape, torch.float32, "tanh", 3, give=lambda t: t.cuda())
    assert torch.equal(plain[0], check(shape, torch.float32, "tanh", 3)[0])

    def sliced(t):
        wide = torch.zeros(t.size(0) + 1, t.size(1) + 2, *t.shape[2:], device="cuda", dtype=t.dtype)
        wide[1:, 1:-1] = t.cuda()
        return wide[1:, 1:-1].detach()

    def off(t):
        flat = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)[1:]
        out = flat.view(t.size(0), *t.shape[2:], t.size(1)).movedim(-1, 1)
        out.copy_(t)
        return out.detach()
    for dtype in TYPES:
        check(shape, dtype, "tanh", 3, give=sliced)
        check(shape, dtype, "tanh", 3, give=off)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_parameters_of_the_activations_type(cuda, lib, dtype):
    check((3, 24, 4, (6, 5)), dtype, "silu", 4, ptype=dtype)


@gpu
def test_without_parameters_and_with_one_of_them(cuda, lib):
    check((3, 24, 4, (6, 5)), torch.float32, "silu", 4, params=False)
    x, w, b, g = make((3, 24, 4, (6, 5)), torch.float32, 4)
    one = torch.ones(24)
    full = L.group_norm(last(x), 4, one.cuda(), b.cuda())
    assert torch.equal(full, L.group_norm(last(x), 4, None, b.cuda()))
    wd = w.cuda().requires_grad_()
    y = L.group_norm(last(x), 4, wd, None, activation="tanh")
    y.backward(last(g))                                      # x itself needs no gradient
    want, most = reference(x, w, torch.zeros(24), 4, "tanh", g)
    assert_within(wd.grad, want[2], most[2], "grad_weight")


@gpu
def test_far_from_zero(cuda, lib):
    """A mean of 1000 times the spread costs the rounding of the mean, not the variance."""
    check((2, 32, 4, (20, 20)), torch.float32, "identity", 6, level=1000.0, spread=1.0)


@gpu
def test_constant_groups_and_values_that_are_not_finite(cuda, lib):
    x = torch.full((2, 8, 5), 7.0, device="cuda")
    y = L.group_norm(x, 2, bias=torch.arange(8.0, device="cuda"))
    assert torch.equal(y, torch.arange(8.0, device="cuda").view(1, 8, 1).expand(2, 8, 5))
    x = torch.randn(2, 8, 5, generator=torch.Generator().manual_seed(1)).cuda()
    clean = L.group_norm(x, 2, activation="relu")
    for bad in (float("inf"), float("nan")):
        x[1, 2, 3] = bad
        y = L.group_norm(x, 2, activation="relu")
        assert torch.isnan(y[1, :4]).all() and torch.equal(y[0], clean[0]) and torch.equal(y[1, 4:], clean[1, 4:])
    empty = torch.zeros(0, 8, 5, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    L.group_norm(empty, 2, w).sum().backward()
    assert empty.grad.shape == (0, 8, 5) and not w.grad.any()


@gpu
def test_same_bits_each_time(cuda, lib):
    x, w, b, g = make((4, 64, 8, (40, 40)), torch.bfloat16, 9)
    runs = [check((4, 64, 8, (40, 40)), torch.bfloat16, "silu", 9) for _ in range(3)]
    for other in runs[1:]:
        assert all(torch.equal(a, e) for a, e in zip(runs[0], other))


@gpu
@pytest.mark.parametrize("shape", [(7, 512, 16, ()), (3, 24, 4, (6, 5)), (1, 16, 2, (150, 150))], ids=ids)
def test_parameters_off_a_boundary_and_twice_backward(cuda, lib, shape):
    """A weight and a bias that lie off a 16-byte boundary; a graph that is gone through twice; a call without gradients."""
    x, w, b, g = make(shape, torch.float32, 12)
    xd = last(x).requires_grad_()
    off = torch.zeros(2, shape[1] + 1, device="cuda")
    off[0, 1:], off[1, 1:] = w.cuda(), b.cuda()
    wo, bo = (off[k, 1:].detach().requires_grad_() for k in range(2))
    wd, bd = w.cuda().requires_grad_(), b.cuda().requires_grad_()
    assert wo.data_ptr() % 16 != 0 or bo.data_ptr() % 16 != 0
    y, want = (L.group_norm(xd, shape[2], *p, activation="silu") for p in ((wo, bo), (wd, bd)))
    first = torch.autograd.grad(y, (xd, wo, bo), last(g), retain_graph=True)
    again = torch.autograd.grad(y, (xd, wo, bo), last(g))
    assert torch.equal(y, want)
    for a, e, f in zip(first, again, torch.autograd.grad(want, (xd, wd, bd), last(g))):
        assert torch.equal(a, e) and torch.equal(a, f)
    with torch.no_grad():
        assert torch.equal(L.group_norm(xd, shape[2], wo, bo, activation="silu"), y)


@gpu
@pytest.mark.parametrize("shape", [(7, 64, 4, ()), (3, 24, 4, (6, 5)), (1, 16, 2, (150, 150))], ids=ids)
def test_dropped_values_are_zero_whatever_they_were(cuda, lib, shape):
    """Infinities make their group's values NaN; dropped ones among them are 0, in the value and in the gradient that reaches dy."""
    x, w, b, g = make(shape, torch.float32, 13)
    x[0, 0] = float("inf")
    rng = torch.tensor([9, 1], dtype=torch.int64, device="cuda")
    y = L.group_norm(last(x), shape[2], w.cuda(), b.cuda(), rate=0.5, rng=rng).cpu()
    kept = numbered(x.shape, 9, 1, 0.5) != 0
    group = torch.zeros(x.shape, dtype=torch.bool)
    group[0, :shape[1] // shape[2]] = True
    assert not y[~kept].any() and torch.isnan(y[kept & group]).all() and torch.isfinite(y[~group]).all()
    none = L.group_norm(last(x), shape[2], rate=1.0, rng=rng)
    assert not none.any()


@gpu
def test_second_derivative_is_refused(cuda, lib):
    x = torch.randn(2, 8, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(L.group_norm(x, 2).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@gpu
def test_streams_and_graphs(cuda, lib):
    """Two streams at once, and a captured forward and backward replayed on new data, give what single calls give."""
    shape = (2, 64, 8, (16, 16))
    data = [make(shape, torch.float32, s) for s in range(4)]

    def step(x, w, b, g):
        y = L.group_norm(x, 8, w, b, activation="silu")
        lo, up = L.group_norm_bound(x - 0.1, x + 0.1, 8, w, b, activation="tanh")
        return [y, lo, up, *torch.autograd.grad([y, lo, up], (x, w, b), [g, g, g])]

    dev = [[last(t) if t.dim() > 1 else t.cuda() for t in d] for d in data]
    for d in dev:
        for t in d[:3]:
            t.requires_grad_()
    single = [step(*d) for d in dev]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    together = []
    for d, s in zip(dev, streams):
        with torch.cuda.stream(s):
            together.append(step(*d))
    torch.cuda.synchronize()
    for a, e in zip(together, single):
        assert all(torch.equal(p, q) for p, q in zip(a, e))
    static = [t.detach().clone().requires_grad_(t.requires_grad) for t in dev[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for gr in graphs:                                         # two graphs, each with scratch of its own
        with torch.cuda.graph(gr):
            outs.append(step(*static))
    for d, e in zip(dev, single):
        with torch.no_grad():
            for t, v in zip(static, d):
                t.copy_(v)
        for gr, out in zip(graphs, outs):
            gr.replay()
            assert all(torch.equal(p, q) for p, q in zip(out, e))


@gpu
def test_more_values_than_32_bits_count(cuda, lib):
    """2^32 + elements: the last sample's values and gradient are those of that sample alone."""
    N, C, side = 2, 64, 5800
    x = torch.empty(N, side, side, C, device="cuda", dtype=torch.float16).permute(0, 3, 1, 2)
    one = last(torch.randn(1, C, 29, 29, generator=torch.Generator().manual_seed(3)).half())
    x.view(N, C, side, side)[:, :, :, :] = one.repeat(1, 1, 200, 200)
    assert x.numel() > 2 ** 32
    w = torch.ones(C, device="cuda").requires_grad_()
    y = L.group_norm(x, 8, w, activation="silu")
    assert torch.equal(y[0], y[1])
    assert_within(y[1, :, -29:, -29:].unsqueeze(0), R.group_norm(one.cpu().double(), 8, None, None, EPS, "silu"), torch.tensor(2e-3), "values")


# ---- the interval form ----------------------------------------------------------------------------------------------------


def make_box(shape, seed, radius, level=3.0):
    x, w, b, g = make(shape, torch.float32, seed, level=level)
    gen = torch.Generator().manual_seed(seed + 1)
    lo = x - radius * torch.rand(x.shape, generator=gen)
    up = x + radius * torch.rand(x.shape, generator=gen)
    w = torch.where(torch.rand(w.shape, generator=gen) < 0.3, -w, w)             # some weights exchange the ends
    return x, lo, up, w, b, g, torch.randn(x.shape, generator=gen)


def bound_reference(lo, up, w, b, groups, act, g0, g1):
    """Values and gradients in 64 bits, and what they may be off by.

    Values: the sums and what a group shares are 64-bit, rounded to fp32 (E; the means in two parts, as good as exact).  n = (l - mean) + own with
    own = (u - l) / M: a rounding of the first difference and one of its second part (2 E |l - mean|, which is at most |n| + |own|), three of
    own, one of the sum: below 4 E (|n| + 2 |own|).  z = n s: that times s, and 2 E |z|.  v = w z + b: |w| times that and E |v|, twice for
    the squares left out.  Then the activation's own error.  Gradients: computed in 64 bits but for v rounded to fp32, the slope
    (norm_reference.error_of_slope of that rounding), its product with the gradient, and one rounding of each result; what a gradient's
    terms may be off by passes through the linear steps behind them by the terms' sizes."""
    leaves = [t.double().requires_grad_() for t in (lo, up, w, b)]
    ys = R.group_norm_bound(*leaves[:2], groups, *leaves[2:], EPS, act)
    grads = torch.autograd.grad(ys, leaves, [g0.double(), g1.double()])
    with torch.no_grad():
        v = R.bound_parts(*[t.double() for t in (lo, up)], groups, w.double(), b.double(), EPS)
        N, C = lo.shape[:2]
        l, u = (t.double().reshape(N, groups, -1) for t in (lo, up))
        M = l.size(2)
        ctr, rad = (l + u) / 2, (u - l) / 2
        sd = ((ctr - ctr.mean(2, keepdim=True)) ** 2).mean(2, keepdim=True).sqrt()
        tight = ((sd - (rad ** 2).mean(2, keepdim=True).sqrt()).clamp(min=0) ** 2 + EPS) ** -0.5
        wide = [(l - u.mean(2, keepdim=True)).abs(), (u - l.mean(2, keepdim=True)).abs()]
        cut = torch.tensor(math.sqrt(M - 1), dtype=torch.float64)
        ez = [4 * E * (n + 3 * rad * 2 / M) * tight + 2 * E * torch.minimum(n * tight, cut) for n in wide]
        ez = torch.maximum(*ez).reshape(lo.shape) * w.double().abs().view([1, C] + [1] * (lo.dim() - 2))
        off = [2 * (ez + E * t.abs()) for t in v]
        most = []
        for y, e, o in zip(ys, v, off):
            worst = torch.maximum(*[R.error_of_act(t, f, act) for t, f in zip(v, off)]) if act == "silu" else R.error_of_act(e, o, act)
            most.append(worst + R.rounded(y, torch.float32))
    # one gradient at a time, its size in the place of its value: d / dv is scaled by what the slope may be off by
    def spread(which, g):
        e = v[which].clone().requires_grad_()
        slope, = torch.autograd.grad(R.activate(e, act).sum(), e)
        off = R.error_of_slope(v[which], E * v[which].abs(), act) + 4 * E * slope.abs()
        return g.double().abs() * off
    off = [spread(k, g) for k, g in enumerate((g0, g1))]
    N, C = lo.shape[:2]
    with torch.no_grad():
        c = [1, C] + [1] * (lo.dim() - 2)
        l, u = (t.double().reshape(N, groups, -1) for t in (lo, up))
        M = l.size(2)
        mean = lambda t: t.mean(2, keepdim=True)  # noqa: E731
        ctr, rad = (l + u) / 2, (u - l) / 2
        ctr = ctr - mean(ctr)
        sd, rho = mean(ctr ** 2).sqrt(), mean(rad ** 2).sqrt()
        tight = ((sd - rho).clamp(min=0) ** 2 + EPS) ** -0.5
        n = torch.maximum((l * (M - 1) - (u.sum(2, keepdim=True) - u)).abs(), (u * (M - 1) - (l.sum(2, keepdim=True) - l)).abs()) / M
        q = ((off[0] + off[1]) * w.double().abs().view(c)).reshape(l.shape)
        d = mean(q * n) * tight ** 3 * (sd + rho)
        gx = (q * tight + mean(q * tight) + d * (ctr.abs() / sd.clamp(min=1e-30) + rad / rho.clamp(min=1e-30))).reshape(lo.shape)
        over = [k for k in range(lo.dim()) if k != 1]
        z = torch.minimum(n * tight, torch.tensor(math.sqrt(M - 1), dtype=torch.float64)).reshape(lo.shape)
        # sums over samples and positions: each partial sum is kept in fp32
        gw = ((off[0] + off[1]) * z).sum(over) + 2 * E * ((g0.double().abs() + g1.double().abs()) * 1.1 * z).sum(over)
        gb = (off[0] + off[1]).sum(over) + 2 * E * ((g0.double().abs() + g1.double().abs()) * 1.1).sum(over)
        most += [gx + R.rounded(grads[0], torch.float32), gx + R.rounded(grads[1], torch.float32), gw + R.rounded(grads[2], torch.float32),
                 gb + R.rounded(grads[3], torch.float32)]
    return [*[y.detach() for y in ys], *grads], most


@gpu
@pytest.mark.parametrize("act", ["identity", "tanh", "silu"])
@pytest.mark.parametrize("radius", [0.01, 1.0], ids=["narrow", "wide"])
@pytest.mark.parametrize("shape", SHAPES, ids=ids)
def test_bounds_and_their_gradients(cuda, lib, shape, radius, act):
    x, lo, up, w, b, g0, g1 = make_box(shape, sum(shape[:3]), radius)
    want, most = bound_reference(lo, up, w, b, shape[2], act, g0, g1)
    leaves = [last(lo).requires_grad_(), last(up).requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()]
    ys = L.group_norm_bound(leaves[0], leaves[1], shape[2], *leaves[2:], eps=EPS, activation=act)
    got = [*ys, *torch.autograd.grad(ys, leaves, [last(g0), last(g1)])]
    for a, e, m, what in zip(got, want, most, ("lower", "upper", "grad_lower", "grad_upper", "grad_weight", "grad_bias")):
        assert_within(a, e, m, what)


@gpu
@pytest.mark.parametrize("act", ["identity", "relu", "tanh", "silu"])
def test_bounds_hold(cuda, lib, act):
    """Values of points in the box, its corners among them, lie within the bounds, up to the roundings of both."""
    for shape in ((3, 24, 4, (6, 5)), (4, 512, 16, ()), (2, 10, 5, (3,))):
        for radius in (0.02, 0.5, 4.0):
            x, lo, up, w, b, _, _ = make_box(shape, 21, radius)
            y0, y1 = L.group_norm_bound(last(lo), last(up), shape[2], w.cuda(), b.cuda(), EPS, act)
            y0, y1 = y0.cpu().double(), y1.cpu().double()
            gen = torch.Generator().manual_seed(5)
            room = 8 * E * (1 + torch.maximum(y0.abs(), y1.abs()))
            for k in range(40):
                t = torch.rand(x.shape, generator=gen)
                y = R.group_norm((lo + (up - lo) * (t.round() if k % 2 else t)).clamp(lo, up).double(), shape[2], w.double(), b.double(), EPS, act)
                assert (y >= y0 - room).all() and (y <= y1 + room).all(), (shape, radius)


@gpu
def test_box_of_one_point(cuda, lib):
    """lower = upper: both bounds are the value, and the gradients add up to the value's."""
    for act in ("identity", "tanh", "silu"):
        shape = (3, 24, 4, (6, 5))
        x, w, b, g = make(shape, torch.float32, 11)
        want, most = reference(x, w, b, 4, act, g)
        leaves = [last(x).requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()]
        for weights in ((1.0, 0.0), (0.0, 1.0)):
            ys = L.group_norm_bound(leaves[0], leaves[0], 4, *leaves[1:], eps=EPS, activation=act)
            got = [sum(k * y for k, y in zip(weights, ys)), *torch.autograd.grad(ys, leaves, [k * last(g) for k in weights])]
            for a, e, m, what in zip(got, want, most, ("value", "grad_x", "grad_weight", "grad_bias")):
                assert_within(a, e, m, what)


@gpu
def test_bound_gradients_against_differences(cuda, lib):
    """The kernel's gradient against differences of the kernel's own values along a direction: with a step of 2^-8 the values' roundings
    (2^-24 of values below 8, 384 of them) and the second derivative's part stay below the tolerance by the sums' sizes."""
    x, lo, up, w, b, g0, g1 = make_box((2, 32, 4, (3,)), 3, 0.3)
    d = torch.randn(lo.shape, generator=torch.Generator().manual_seed(8))
    a = [last(t) for t in (lo, up, d, g0, g1)]
    lod, upd = a[0].requires_grad_(), a[1].requires_grad_()
    f = lambda s: sum((y.double() * g.double()).sum() for y, g in zip(L.group_norm_bound(lod + s * a[2], upd + s * a[2], 4, w.cuda(), b.cuda()), a[3:]))  # noqa: E731
    gl, gu = torch.autograd.grad(f(0.0), (lod, upd))
    with torch.no_grad():
        h = 2.0 ** -8
        third = ((f(h) - f(-h)) / (2 * h) - (f(h / 2) - f(-h / 2)) / h).abs()          # what a finer step still changes
        slope = (f(h / 2) - f(-h / 2)) / h
        rounding = 384 * 2.0 ** -21 * 4 / h
    assert abs(((gl + gu) * a[2]).sum().double() - slope) <= third + rounding


@gpu
def test_bounds_off_a_boundary_and_not_finite(cuda, lib):
    x, lo, up, w, b, _, _ = make_box((3, 24, 4, (6, 5)), 3, 0.1)
    want = L.group_norm_bound(last(lo), last(up), 4, w.cuda(), b.cuda())
    flat = torch.empty(lo.numel() + 1, device="cuda")[1:].view(3, 6, 5, 24).permute(0, 3, 1, 2)
    flat.copy_(lo)
    got = L.group_norm_bound(flat, last(up), 4, w.cuda(), b.cuda())
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    up[1, 2, 3, 4] = float("inf")
    got = L.group_norm_bound(last(lo), last(up), 4, w.cuda(), b.cuda())
    assert all(torch.isnan(p[1, :6]).all() and torch.equal(p[0], q[0]) and torch.equal(p[1, 6:], q[1, 6:]) for p, q in zip(got, want))


# ---- as a user has them together ------------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("shape", [(7, 64, 4, ()), (3, 24, 4, (6, 5)), (1, 16, 2, (150, 150))], ids=ids)
def test_boxes_wider_than_their_type(cuda, lib, shape):
    """Boxes whose width leaves fp32: every normalised value is possible, so the bounds are -+sqrt(M - 1), where they are cut."""
    n, c, groups, space = shape
    l = last(torch.full((n, c, *space), -3e38))
    lo, up = L.group_norm_bound(l, -l, groups)
    m = c // groups * math.prod(space)
    # the root is rounded once, from M - 1 < 2^24
    assert torch.allclose(up, torch.full_like(up, math.sqrt(m - 1)), rtol=2.0 ** -23, atol=0) and torch.equal(lo, -up)


@gpu
@pytest.mark.parametrize("groups, dropout", [(None, 0.25), (4, 0.0), (4, 0.25)])
def test_head_on_a_triple(cuda, lib, groups, dropout):
    """The head with its norm and dropout: the same values as the plain implementations step by step, the value within its bounds,
    gradients for every parameter."""
    torch.manual_seed(3)
    head = L.Predictor(32, 16, 5, groups=groups, dropout=dropout).cuda().train()
    x = torch.randn(20, 32, device="cuda")
    t = torch.randint(0, 5, (20,), device="cuda")
    module = head.norm if groups else head.drop
    before = module.rng.tolist() if dropout else None
    y, worst = head(x, x - 0.05, x + 0.05, targets=t)
    (y.sum() + worst.clamp(min=0).sum()).backward()
    assert all(q.grad is not None and torch.isfinite(q.grad).all() for q in head.parameters())
    triple = [v.double().cpu() for v in head.fc1(x, x - 0.05, x + 0.05)]
    if groups:
        w, b = head.norm.weight.detach().cpu().double(), head.norm.bias.detach().cpu().double()
        value = R.group_norm(triple[0], groups, w, b, 1e-5, "tanh")
        lo, up = R.group_norm_bound(*triple[1:], groups, w, b, 1e-5, "tanh")
    else:
        value, lo, up = map(torch.tanh, triple)
    if dropout:
        factor = numbered((20, 16), *before, dropout)
        value, lo, up = value * factor, lo * factor, up * factor
        assert module.rng.tolist() == [before[0], before[1] + 1]
    assert (lo <= value).all() and (value <= up).all()
    with torch.no_grad():
        wanted = head.fc2(value.float().cuda(), lo.float().cuda(), up.float().cuda(), targets=t)
    for a, e in zip((y, worst), wanted):
        assert (a - e).abs().max() < 1e-4 * (1 + e.abs().max())
    head.eval()
    twice = [head(x, x - 0.05, x + 0.05, targets=t) for _ in range(2)]
    assert all(torch.equal(a, e) for a, e in zip(*twice))


@gpu
def test_training_and_certification_of_a_net(cuda, lib):
    """A '++' net with a normalised head takes training steps, and its certificates hold for attacked inputs."""
    torch.manual_seed(5)
    feature = L.MLPFeature(2, 1, 64)
    net = L.Model(feature, L.Predictor(feature.out_features, 32, 4, groups=4, dropout=0.1), 0.02).cuda()
    L.set_p_norm(net, float("inf"))
    from linfdist_b200.train_step import DataParallelStep, MarginLoss, cross_entropy
    opt = L.AdamW(net, lr=0.01)
    step, loss = DataParallelStep(net, opt), MarginLoss(cross_entropy(), 0.75)
    x, t = torch.rand(48, 64, device="cuda"), torch.randint(0, 4, (48,), device="cuda")
    start = [q.detach().clone() for q in net.parameters()]
    net.train()
    for _ in range(3):
        out, worst = step(x, targets=t)
        opt.zero_grad(set_to_none=True)
        loss(out, worst, t).backward()
        step.finish_step()
    step.synchronize()
    assert all(torch.isfinite(q).all() and not torch.equal(q, s) for q, s in zip(net.parameters(), start))
    one, zero = torch.ones((), device="cuda"), torch.zeros((), device="cuda")
    net.eval()
    ok, margins = L.certify(net, x, t, 1e-3, one, zero)
    again = L.certify(net, x, t, 1e-3, one, zero, values=True)
    assert torch.equal(margins, again[1])
    bad = L.AttackPGD(net, 1e-3, 5e-4, 3, one, zero).find(x, t)
    with torch.no_grad():
        logits = net(bad)
    attained = logits - logits.gather(1, t.view(-1, 1))
    assert (attained <= margins + 1e-4 * (1 + margins.abs())).all()
    assert (logits.argmax(1) == t)[ok].all()


@gpu
def test_behind_a_convolution(cuda, lib):
    """Distance convolution -> group norm -> dropout -> distance convolution: the channels stay last in memory up to the second
    convolution, and the values and gradients are those of the same chain on plain memory."""
    torch.manual_seed(6)
    p = float("inf")
    first = L.NormDistConv(4, 32, 3, padding=1, p=p, channels_last=True).cuda()
    norm = L.BoundGroupNorm(8, 32, activation="silu").cuda()
    drop = L.BoundDropout(0.2, seed=9).cuda()
    second = L.NormDistConv(32, 32, 3, padding=1, p=p).cuda()
    x = torch.randn(2, 4, 8, 8, device="cuda")
    results = []
    for last_too in (True, False):
        first.channels_last = last_too
        drop.rng[1] = 0
        xl = x.clone().requires_grad_()
        y = first(xl)[0]
        assert y.is_contiguous(memory_format=torch.channels_last) == last_too
        z = drop(norm(y)[0])[0]
        assert z.is_contiguous(memory_format=torch.channels_last)
        out = second(z)[0]
        grads = torch.autograd.grad(out.square().sum(), [xl, *first.parameters(), *norm.parameters(), *second.parameters()])
        results.append([out, *grads])
    assert all(torch.equal(a, e) for a, e in zip(*results))
