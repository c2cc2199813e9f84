"""Group norm, its interval form and their gradients where arithmetic runs out: long columns, values far from 0, values at the ends of
their type.  Everything is compared with the formulas in 64 bits; the tolerances are worked out beside the tests."""
import math

import pytest
import torch

import linfdist_b200 as L
import norm_reference as R
from norm_reference import E

gpu = pytest.mark.gpu
EPS = 1e-5


def stored(N, C, L_, dtype, seed, spread=0.5, level=3.0):
    """[N, C, L_] on the GPU, the channels last in memory."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(N, L_, C, generator=gen, device="cuda").mul_(spread).add_(level)
    return x.to(dtype).movedim(-1, 1)


def parts(x, groups):
    """(h, mean, 1 / deviation) of [N, C, L] in 64 bits on the device of x, h as [N, groups, C / groups, L]."""
    t = x.detach().double().view(x.size(0), groups, x.size(1) // groups, -1)
    mean = t.mean((2, 3), keepdim=True)
    t = t - mean
    r = (t.square().mean((2, 3), keepdim=True) + EPS).rsqrt()
    return t.mul_(r), mean, r


def assert_within(got, want, most, what):
    bad = ~((got.double() - want).abs() <= most)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got.double() - want).abs() - most).max():.3g} over"


# (N, C, groups, positions, rows of threads): the two passes with 2048 and 512 rows to a thread, vectors within one group and across several;
# the kept form; elements one by one
LONG = [(1, 1024, 32, 131072, 64), (1, 1024, 512, 131072, 64), (1, 255, 1, 32768, 64), (3, 8, 2, 2000, 128), (3, 12, 12, 1000, 85)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", LONG, ids=lambda c: "C{}_G{}_L{}".format(*c[1:4]))
def test_first_rows_apart_from_the_rest(cuda, lib, case, dtype):
    """Every thread's first row lies 300 deviations off (a border, a special position).

    A thread's first run has 8 rows, seven of them D off the shift.  Their sums are off by 7 E of 7 D and 7 D^2, so their sum of squares about
    their mean by less than 135 E D^2; the runs behind it stand D / 8 off their shift at most and add less than 50 E D^2, the later ones 2.
    The thread's own sum of squares is at least D^2 (1 - 1 / n), so the variance is off by less than 200 E of itself, 1 / deviation by
    100 E.  The mean: 49 E D of the first run and 128 E D of the second, over n values, with D at most sqrt(n) deviations: below 177 E / sqrt(n)
    deviations.  Then the roundings of the element itself."""
    N, C, groups, n, first = case
    x = stored(N, C, n, dtype, sum(case))
    x[:, :, :first] += 150.0
    y = L.group_norm(x, groups, eps=EPS)
    h, mean, r = parts(x, groups)
    most = 100 * E * h.abs() + 177 * E / math.sqrt(n / first) + 6 * E * (h.abs() + r * mean.abs()) + R.HALF_STEP[dtype] * h.abs() + 1e-30
    assert_within(y.view(h.shape), h, most, "values")


# dense; kept, vectors within one group and across several; the two passes, both as well
FAR = [(7, 512, 16, 1), (5, 64, 8, 9), (3, 24, 4, 30), (2, 2, 1, 50), (1, 64, 8, 40000), (1, 24, 4, 22500), (2, 3, 1, 9000)]


@gpu
@pytest.mark.parametrize("case", FAR, ids=lambda c: "N{}_C{}_G{}_L{}".format(*c))
def test_values_very_far_from_zero(cuda, lib, case):
    """A mean of 10^6 deviations: the mean is not rounded to fp32 anywhere, so the values are off by their own roundings alone and lie within the bounds
    of a box of one point.

    x less the mean's first part is exact (both are fp32 numbers less than a factor of two apart); the second part goes into the added
    term, which is below 2^-24 * 10^6 / deviation and rounded once; 1 / deviation, its product with the difference, the sum: E each.  Parts of the sums
    are joined about one shift, off by a few roundings of a deviation, as the variance is by a few of its own: 16 E in all."""
    N, C, groups, n = case
    x = stored(N, C, n, torch.float32, sum(case), level=5e5)
    x = x if n > 1 else x.reshape(N, C)
    h, mean, r = parts(x, groups)
    most = 16 * E * (1 + h.abs()) + E * E * r * mean.abs()
    y = L.group_norm(x, groups, eps=EPS)
    assert_within(y.reshape(h.shape), h, most, "values")


# (N, C, groups, positions, additions in a row before: the gradient below is the one that many of them lose most with)
CONSTANT = [(1, 1024, 32, 131072, 2048), (1, 255, 5, 300000, 2048), (444 * 256 * 512, 8, 1, 1, 512)]


@gpu
@pytest.mark.parametrize("case", CONSTANT, ids=lambda c: "N{}_C{}_G{}_L{}".format(*c[:4]))
def test_constant_gradients_over_long_columns(cuda, lib, case):
    """A gradient that is the same everywhere: every addition in a row rounds the same way, by up to half a step.

    64 additions of equal terms in fp32 are off by at most E (64 + 1) / 2 of the sum; the partial sum is rounded once before 64-bit sums take over, and
    so is the result: 36 E of the terms' sizes.  The weight's terms have h, off by 10 E (1 + |h|) of itself, besides."""
    N, C, groups, n, adds = case
    c = 1 + 0.499 * 2.0 ** (math.log2(adds) - 24)
    x = stored(N, C, n, torch.float32, sum(case) % 1000)
    x = (x if n > 1 else x.reshape(N, C)).requires_grad_()
    w, b = torch.ones(C, device="cuda", requires_grad=True), torch.zeros(C, device="cuda", requires_grad=True)
    y = L.group_norm(x, groups, w, b, EPS)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.full_like(y, c))
    del y, gx
    c = torch.tensor(c).double().item()          # as fp32 has it
    assert_within(gb, torch.full((C,), N * n * c, dtype=torch.float64, device="cuda"), 36 * E * N * n * c, "grad_bias")
    h = parts(x.view(N, C, n), groups)[0].view(N, C, n)
    assert_within(gw, c * h.sum((0, 2)), c * ((36 + 10) * E * h.abs().sum((0, 2)) + 10 * E * N * n), "grad_weight")


# (N, C, groups, positions): dense, kept, kept with vectors across groups, the two passes
EDGE = [(1, 4, 1, 1), (3, 64, 4, 1), (2, 24, 4, 30), (2, 24, 12, 30), (1, 16, 2, 22500)]


@gpu
@pytest.mark.parametrize("act", ["identity", "tanh"])
@pytest.mark.parametrize("case", EDGE, ids=lambda c: "N{}_C{}_G{}_L{}".format(*c))
def test_boxes_at_the_edge_of_fp32(cuda, lib, case, act):
    """Values whose distance from their mean is beyond fp32: the bounds are ordered and those of the formulas.

    The differences are taken in 64 bits, 1 / deviation is a normal number (2^64 times as large): each rounded once, their product once, then a
    bound's own roundings: 8 E of it (weights 1, biases 0), and tanhf's 4 E."""
    N, C, groups, n = case
    gen = torch.Generator().manual_seed(sum(case))
    x = 3e38 * torch.where(torch.rand(N, C, n, generator=gen) < 0.25, 1.0, -1.0)
    x[:, ::C // groups, 0] = 3e38                    # one at least in each group, and one that is not
    x[:, C // groups - 1::C // groups, n - 1] = -3e38
    lo, up = x, (x.double() + 1e37 * torch.rand(x.shape, generator=gen).double()).float()
    if n == 1:
        lo, up = lo[..., 0], up[..., 0]
    for low, high in ((lo, up), (lo, lo)):
        want = R.group_norm_bound(low.double(), high.double(), groups, None, None, EPS, act)
        got = [t.cpu() for t in L.group_norm_bound(low.cuda(), high.cuda(), groups, eps=EPS, activation=act)]
        assert torch.isfinite(got[0]).all() and (got[0] <= got[1]).all()
        for g, w, what in zip(got, want, ("lower", "upper")):
            assert_within(g, w, 12 * E * w.abs() + 8 * E * (1 if act == "tanh" else 0), what)


@gpu
@pytest.mark.parametrize("case", FAR, ids=lambda c: "N{}_C{}_G{}_L{}".format(*c))
def test_boxes_very_far_from_zero(cuda, lib, case):
    """Boxes around values of 10^6 deviations: the deviation is that of the formulas, the bounds are ordered, and a value is within the bounds of its own
    box.

    The 64-bit squares are taken about a value of the group, so 1 / deviation is as good as exact before it is rounded: E.  Differences from a
    mean in two parts, twice rounded, own three times; the product: 12 E (1 + |bound|), with n below 2 |bound| + 1 deviations of the centres."""
    N, C, groups, n = case
    lo = stored(N, C, n, torch.float32, sum(case), level=5e5)
    up = lo + 0.0625 * torch.randint(0, 3, lo.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    if n == 1:
        lo, up = lo.reshape(N, C), up.reshape(N, C)
    for low, high in ((lo, up), (lo, lo)):
        one = torch.ones(C, dtype=torch.float64, device="cuda")
        want = R.group_norm_bound(low.double(), high.double(), groups, one, 0 * one, EPS, "identity")
        got = L.group_norm_bound(low, high, groups, eps=EPS)
        assert (got[0] <= got[1]).all()
        for g, w, what in zip(got, want, ("lower", "upper")):
            assert_within(g, w, 12 * E * (1 + w.abs()), what)
    value = L.group_norm(lo, groups, eps=EPS)
    room = 28 * E * (1 + value.abs())                       # 16 of the value, 12 of the bound
    assert (got[0] - room <= value).all() and (value <= got[1] + room).all()


@gpu
@pytest.mark.parametrize("case", [(1, 1024, 32, 131072, 1024), (148 * 6 * 300, 64, 4, 2, 256)], ids=lambda c: "N{}_C{}_G{}_L{}".format(*c[:4]))
def test_constant_gradients_of_boxes_over_long_columns(cuda, lib, case):
    """As above, for the parameters of the bounds: 64-bit sums of a CTA's rows and samples, rounded once (E), then 64-bit sums, rounded once; the slope's
    product with the gradient is exact here.  The weight's terms have z, which is that of the formulas, to 64 bits."""
    N, C, groups, n, adds = case
    c = (1 + 0.499 * 2.0 ** (math.log2(adds) - 24)) / 2
    lo = stored(N, C, n, torch.float32, sum(case) % 1000)
    up = lo + 0.01
    w, b = torch.ones(C, device="cuda", requires_grad=True), torch.zeros(C, device="cuda", requires_grad=True)
    ys = L.group_norm_bound(lo, up, groups, w, b, EPS)
    g = torch.full_like(lo, c)
    gw, gb = torch.autograd.grad(ys, (w, b), (g, g))
    c = torch.tensor(c).double().item()
    assert_within(gb, torch.full((C,), 2 * N * n * c, dtype=torch.float64, device="cuda"), 3 * E * 2 * N * n * c, "grad_bias")
    z = sum(y.detach().double() for y in ys)                   # fp32, off by less than 12 E (1 + |z|) each
    size = sum((y.detach().double().abs() + 1).sum((0, 2)) for y in ys)
    assert_within(gw, c * z.sum((0, 2)), c * 16 * E * size, "grad_weight")


@gpu
@pytest.mark.parametrize("case", FAR + [(2, 8192, 1, 1), (1, 2048, 1, 4096)], ids=lambda c: "N{}_C{}_G{}_L{}".format(*c))
def test_values_as_far_apart_as_the_header_allows(cuda, lib, case):
    """Values 10^15 from each other (their squares by the thousand are far beyond what one square would say), and equal ones of 10^37.

    As for far values: 16 E (1 + |h|); the gradient is 1 / deviation times terms of order 1 that are off by 16 E each, and by 36 E in their means."""
    N, C, groups, n = case
    x = stored(N, C, n, torch.float32, sum(case), spread=1.0, level=0.0).clamp_(-4, 4).mul_(1.2e14)
    x = (x if n > 1 else x.reshape(N, C)).requires_grad_()
    h, mean, r = parts(x.reshape(N, C, n), groups)
    y = L.group_norm(x, groups, eps=EPS)
    assert_within(y.reshape(h.shape), h, 16 * E * (1 + h.abs()), "values")
    g = torch.randn(y.shape, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    gx, = torch.autograd.grad(y, x, g)
    g = g.double().reshape(h.shape)
    both = lambda t: t.mean((2, 3), keepdim=True)  # noqa: E731
    want = r * (g - both(g) - h * both(g * h))
    most = r * (16 * E * (g.abs() + (1 + h.abs()) * both((1 + h.abs()) * g.abs())) + 36 * E * (both(g.abs()) + h.abs() * both((g * h).abs())))
    assert_within(gx.reshape(h.shape), want, most, "grad_x")
    assert not L.group_norm(torch.full_like(x, 1e37), groups).any()
