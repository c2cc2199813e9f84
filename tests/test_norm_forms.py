"""Forms of the norms and of dropout beside those of test_group_norm.py and test_dropout.py: relu's gradients, layouts of boxes, triples of 16 bits,
gradients beyond 2^32 elements."""
import pytest
import torch

import linfdist_b200 as L
import norm_reference as R
import test_dropout as D
import test_group_norm as T

gpu = pytest.mark.gpu
MAPS = [(5, 30, 3, (5, 7)), (2, 64, 8, (16, 16)), (3, 75, 5, (37,)), (2, 320, 32, (8, 8)), (7, 512, 16, ()), (1, 16, 2, (150, 150))]


def away_from(u, g):
    """g with zeros where relu's slope may jump: |u| is off by far less than 2^-10."""
    return torch.where(u.abs() > 2.0 ** -10, g, torch.zeros((), dtype=g.dtype))


@gpu
@pytest.mark.parametrize("dtype", T.TYPES)
@pytest.mark.parametrize("shape", MAPS, ids=T.ids)
def test_relu_on_maps(cuda, lib, shape, dtype):
    x, w, b, g = T.make(shape, dtype, 17)
    g = away_from(R.norm_parts(x.double(), shape[2], w.double(), b.double(), T.EPS)[3], g)
    want, most = T.reference(x, w, b, shape[2], "relu", g)
    leaves = [T.last(x).requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()]
    y = L.group_norm(leaves[0], shape[2], *leaves[1:], eps=T.EPS, activation="relu")
    for a, e, m, what in zip([y, *torch.autograd.grad(y, leaves, T.last(g))], want, most, ("value", "grad_x", "grad_weight", "grad_bias")):
        T.assert_within(a, e, m, what)


@gpu
@pytest.mark.parametrize("radius", [0.01, 1.0], ids=["narrow", "wide"])
@pytest.mark.parametrize("shape", MAPS, ids=T.ids)
def test_relu_on_bounds(cuda, lib, shape, radius):
    x, lo, up, w, b, g0, g1 = T.make_box(shape, 18, radius)
    v = R.bound_parts(lo.double(), up.double(), shape[2], w.double(), b.double(), T.EPS)
    g0, g1 = (away_from(u, g) for u, g in zip(v, (g0, g1)))
    want, most = T.bound_reference(lo, up, w, b, shape[2], "relu", g0, g1)
    leaves = [T.last(lo).requires_grad_(), T.last(up).requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()]
    ys = L.group_norm_bound(*leaves[:2], shape[2], *leaves[2:], eps=T.EPS, activation="relu")
    got = [*ys, *torch.autograd.grad(ys, leaves, [T.last(g0), T.last(g1)])]
    for a, e, m, what in zip(got, want, most, ("lower", "upper", "grad_lower", "grad_upper", "grad_weight", "grad_bias")):
        T.assert_within(a, e, m, what)


@gpu
def test_bounds_of_plain_memory(cuda, lib):
    """Boxes and gradients in plain NCHW memory, one of each: bit for bit what channels-last ones give."""
    shape = (3, 24, 4, (6, 5))
    x, lo, up, w, b, g0, g1 = T.make_box(shape, 19, 0.1)
    results = []
    for give in ((T.last, T.last, T.last, T.last), [lambda t: t.cuda()] * 4, (T.last, lambda t: t.cuda(), lambda t: t.cuda(), T.last)):
        leaves = [give[0](lo).requires_grad_(), give[1](up).requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()]
        ys = L.group_norm_bound(*leaves[:2], 4, *leaves[2:], activation="tanh")
        results.append([*ys, *torch.autograd.grad(ys, leaves, [give[2](g0), give[3](g1)])])
    for other in results[1:]:
        assert all(torch.equal(a, e) for a, e in zip(results[0], other))


@gpu
@pytest.mark.parametrize("dtype", T.TYPES)
@pytest.mark.parametrize("shape", [(33, 51), (2, 6, 5, 7)])
def test_triples_of_every_type(cuda, lib, shape, dtype):
    gen = torch.Generator().manual_seed(3)
    data = [torch.randn(shape, generator=gen).to(dtype) for _ in range(6)]
    leaves = [t.cuda().requires_grad_() for t in data[:3]]
    out = L.dropout(leaves[0], 0.3, D.state(11, 5), *leaves[1:])
    grads = torch.autograd.grad(out, leaves, [t.cuda() for t in data[3:]])
    for a, e in zip([*out, *grads], data):
        assert D.same(a, D.expected(e, 11, 5, 0.3))


@gpu
def test_gradients_beyond_2_32_values(cuda, lib):
    """2^32 + elements of one tile laid side by side: the last tile's gradient is the tile's, the parameters' 40000 times the tile's.

    fp16 gradients by R.rounded and 2^-9 of 1 / deviation for the sums; the parameters' terms are off by 2^-9 of themselves at most."""
    N, C, side, times = 2, 64, 5800, 200
    gen = torch.Generator().manual_seed(3)
    tile, dtile = (torch.randn(1, C, side // times, side // times, generator=gen).half() for _ in range(2))
    x, g = (torch.empty(N, side, side, C, device="cuda", dtype=torch.float16).permute(0, 3, 1, 2).copy_(T.last(t).repeat(1, 1, times, times)) for t in (tile, dtile))
    assert x.numel() > 2 ** 32
    w, b = torch.ones(C, device="cuda", requires_grad=True), torch.zeros(C, device="cuda", requires_grad=True)
    x.requires_grad_()
    y = L.group_norm(x, 8, w, b, activation="tanh")
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
    del y
    assert torch.equal(gx[0, :, :29, :29], gx[1, :, -29:, -29:])
    want, _ = T.reference(tile, w.detach().cpu(), b.detach().cpu(), 8, "tanh", dtile)
    r = R.norm_parts(tile.double(), 8, None, None, T.EPS)[1]
    T.assert_within(gx[1:, :, -29:, -29:], want[1], r * 2.0 ** -9 + R.rounded(want[1], torch.float16), "grad_x")
    size = dtile.double().abs().sum((0, 2, 3)) * 2.0 ** -9
    h = R.norm_parts(tile.double(), 8, None, None, T.EPS)[2].abs()
    T.assert_within(gw / (N * times ** 2), want[2], (dtile.double().abs() * (1 + h)).sum((0, 2, 3)) * 2.0 ** -9, "grad_weight")
    T.assert_within(gb / (N * times ** 2), want[3], size, "grad_bias")
