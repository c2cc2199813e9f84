"""Dropout whose mask is computed and never stored: bit for bit against the generator in numpy; refusals; streams, graphs, triples."""
import ctypes

import pytest
import torch

import linfdist_b200 as L
import norm_reference as R
from linfdist_b200 import _lib

TYPES = [torch.float32, torch.float16, torch.bfloat16]
gpu = pytest.mark.gpu


def state(seed, offset=0, device="cuda:0"):
    return torch.tensor([seed, offset], dtype=torch.int64, device=device)


def expected(x, seed, offset, rate):
    """x on the CPU, elements numbered as x.reshape(-1) has them: the fp32 product with the fp32 scale, rounded once to the type of x."""
    if R.threshold(rate) == 0:
        return x
    keep = R.kept(seed, offset, x.numel(), rate).view(x.shape)
    return torch.where(keep, x.float() * torch.tensor(R.scale(rate), dtype=torch.float32), torch.zeros(())).to(x.dtype)


def same(a, b):
    a, b = a.detach().cpu().contiguous(), b.detach().cpu().contiguous()
    kind = torch.int32 if a.dtype == torch.float32 else torch.int16
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.view(kind), b.view(kind))


def test_generator_against_published_words():
    """Known answers of Philox4x32 with 7 rounds: all-zero counter and key, all-one counter and key."""
    w = R.pieces(0, 0, 8)
    assert [int(w[2 * i] + 65536 * w[2 * i + 1]) for i in range(4)] == [0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48]


def test_mask_has_the_rate_and_no_pattern():
    n, rate = 1 << 20, 0.3
    a, b = R.kept(5, 0, n, rate).double(), R.kept(5, 1, n, rate).double()
    sd = (rate * (1 - rate) / n) ** 0.5
    assert abs(a.mean() - (1 - rate)) < 5 * sd
    for other in (b, a.roll(1), a.roll(8), a.roll(512)):
        assert abs(((a - 0.7) * (other - 0.7)).mean()) < 5 * rate * (1 - rate) / n ** 0.5


@pytest.mark.parametrize("call, code", [
    (dict(x=None), 1), (dict(y=None), 1), (dict(y_lower=None), 1), (dict(n=0), 2), (dict(n=-5), 2), (dict(type=3), 8), (dict(type=-1), 8),
    (dict(rate=-0.1), 9), (dict(rate=1.5), 9), (dict(rate=float("nan")), 9), (dict(rng=None), 9)])
def test_library_refuses(lib, call, code):
    p = ctypes.c_void_p(4096)          # never followed: each call is refused before a launch
    a = dict(x=p, lower=p, upper=p, n=8, type=0, rate=0.5, rng=p, y=p, y_lower=p, y_upper=p, stream=None)
    a.update(call)
    assert lib.linf_dropout(*a.values()) == code
    assert lib.linf_dropout_next(None, p, None) == 1 and lib.linf_dropout_next(p, None, None) == 1


def test_python_refuses_on_the_host():
    x, rng = torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64)
    for rate in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            L.dropout(x, rate, rng)
        with pytest.raises(ValueError):
            L.BoundDropout(rate)
    for bad in (torch.zeros(2), torch.zeros(3, dtype=torch.int64), torch.zeros(4, dtype=torch.int64)[::2], 7):
        with pytest.raises(RuntimeError, match="rng"):
            L.dropout(x, 0.5, bad)
    with pytest.raises(RuntimeError, match="together"):
        L.dropout(x, 0.5, rng, lower=x)
    with pytest.raises(RuntimeError, match="upper"):
        L.dropout(x, 0.5, rng, lower=x, upper=torch.zeros(3, 2))
    with pytest.raises(RuntimeError, match="lower"):
        L.dropout(x, 0.5, rng, lower=x.double(), upper=x)
    with pytest.raises(RuntimeError, match="CUDA"):
        L.dropout(x, 0.5, rng)
    with pytest.raises(RuntimeError, match="CUDA"):
        L.dropout_next(rng)


def test_module_without_effect_on_the_host():
    """Eval mode and rate 0 give back what came; only a rate above 0 keeps a generator state."""
    x = torch.randn(2, 3)
    drop = L.BoundDropout(0.5, seed=3)
    assert set(drop.state_dict()) == {"rng"} and drop.rng.tolist() == [3, 0]
    assert drop.eval()(x, x - 1, x + 1)[0] is x
    assert L.BoundDropout(0.0).train()(x)[0] is x and not L.BoundDropout(0.0).state_dict()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 255, 2048, 2049, 100003])
@pytest.mark.parametrize("rate", [0.1, 0.5, 1.0])
def test_values_and_gradient(cuda, lib, dtype, n, rate):
    gen = torch.Generator().manual_seed(n)
    x, g = (torch.randn(n, generator=gen).to(dtype) for _ in range(2))
    seed, offset = 0x1234567890ABCDEF, (1 << 40) + 3
    xd = x.cuda().requires_grad_()
    y = L.dropout(xd, rate, state(seed, offset))
    assert same(y, expected(x, seed, offset, rate))
    y.backward(g.cuda())
    assert same(xd.grad, expected(g, seed, offset, rate))


@gpu
def test_rates_at_the_ends(cuda, lib):
    x = torch.tensor([1.0, -2.0, float("inf"), float("nan"), -0.0] * 40, device="cuda")
    assert same(L.dropout(x, 0.0, state(1)), x) and same(L.dropout(x, 2.0 ** -18, state(1)), x)      # a threshold of 0 keeps all as it is
    assert same(L.dropout(x, 1.0, state(1)), torch.zeros_like(x))                                     # also what is infinite or no number
    assert (L.dropout(torch.ones(1 << 16, device="cuda"), 65535 / 65536, state(1)).unique().cpu() == torch.tensor([0.0, 65536.0])).all()
    y = L.dropout(x, 0.5, state(9))
    keep = R.kept(9, 0, x.numel(), 0.5)
    assert not y.cpu()[~keep].any() and torch.isnan(y.cpu()[keep]).sum() == torch.isnan(x.cpu()[keep]).sum()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_offset_and_strides(cuda, lib, dtype):
    """Tensors off a 16-byte boundary, cut out of others, channels last and transposed."""
    base = torch.randn(4, 6, 5, 7, generator=torch.Generator().manual_seed(1)).to(dtype)
    flat = base.reshape(-1).cuda()
    assert same(L.dropout(flat[3:], 0.4, state(7)), expected(base.reshape(-1)[3:], 7, 0, 0.4))
    assert same(L.dropout(base.cuda()[:, 1:4], 0.4, state(7)), expected(base[:, 1:4].contiguous(), 7, 0, 0.4))
    last = base.cuda().to(memory_format=torch.channels_last).requires_grad_()
    y = L.dropout(last, 0.4, state(7))
    want = expected(base.permute(0, 2, 3, 1).contiguous(), 7, 0, 0.4).permute(0, 3, 1, 2)
    assert same(y, want) and y.is_contiguous(memory_format=torch.channels_last)
    g = torch.randn(base.shape, generator=torch.Generator().manual_seed(2)).to(dtype)
    y.backward(g.cuda())                                  # a gradient in another layout than the value
    assert same(last.grad, expected(g.permute(0, 2, 3, 1).contiguous(), 7, 0, 0.4).permute(0, 3, 1, 2))
    wide = torch.randn(3, 1, dtype=torch.float32).to(dtype).cuda().expand(3, 40)
    assert same(L.dropout(wide, 0.4, state(7)), expected(wide.cpu().contiguous(), 7, 0, 0.4))
    assert L.dropout(base.cuda()[:0], 0.4, state(7)).shape == (0, 6, 5, 7)


@gpu
def test_triple_under_one_mask(cuda, lib):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(33, 51, generator=gen)
    lo, up = x - torch.rand(33, 51, generator=gen), x + torch.rand(33, 51, generator=gen)
    t = [v.cuda().requires_grad_() for v in (x, lo, up)]
    out = L.dropout(t[0], 0.3, state(11, 5), t[1], t[2])
    for o, v in zip(out, (x, lo, up)):
        assert same(o, expected(v, 11, 5, 0.3))
    assert (out[1] <= out[0]).all() and (out[0] <= out[2]).all()
    g = torch.randn(33, 51, generator=gen)
    gx, gl, gu = torch.autograd.grad([out[1]], t, [g.cuda()], allow_unused=True)      # the value and the upper bound are not used
    assert gx is None and gu is None and same(gl, expected(g, 11, 5, 0.3))


@gpu
def test_many_elements_number_beyond_32_bits(cuda, lib):
    """Element numbers above 2^32 reach the generator whole."""
    n = (1 << 32) + 4096
    x = torch.ones(n, dtype=torch.float16, device="cuda")
    y = L.dropout(x, 0.5, state(77, 2))
    del x
    first, last = y[:4096].cpu(), y[-4096:].cpu()
    assert same(first, 2.0 * R.kept(77, 2, 4096, 0.5).to(torch.float16))
    keep = R.kept(77, 2, 4096, 0.5, first=1 << 32)
    assert same(last, 2.0 * keep.to(torch.float16)) and not same(first, last)


@gpu
def test_state_draws_each_offset_once(cuda, lib):
    rng = state(5, 40)
    used = [L.dropout_next(rng) for _ in range(3)]
    assert [u.tolist() for u in used] == [[5, 40], [5, 41], [5, 42]] and rng.tolist() == [5, 43]
    x = torch.ones(100, device="cuda", requires_grad=True)
    y = L.dropout(x, 0.5, rng)                   # the state itself, moved on before the backward pass: refused
    L.dropout_next(rng)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


@gpu
def test_two_streams_get_masks_of_their_own(cuda, lib):
    rng = state(5)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    used = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                used.append(L.dropout_next(rng))
    torch.cuda.synchronize()
    assert sorted(u[1].item() for u in used) == list(range(40))


@gpu
def test_captured_graph_draws_anew(cuda, lib):
    drop = L.BoundDropout(0.5, seed=8).cuda().train()
    x = torch.randn(1000, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        drop(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = drop(x)[0]
    before = drop.rng[1].item()
    for k in range(3):
        graph.replay()
        assert same(y, expected(x.cpu(), 8, before + k, 0.5))
    assert drop.rng[1].item() == before + 3


@gpu
def test_gradient_is_the_slope(cuda, lib):
    """Dropout is linear: a difference of values is the gradient's product with the step."""
    gen = torch.Generator().manual_seed(4)
    x, d, g = (torch.randint(-64, 64, (501,), generator=gen).float().cuda() for _ in range(3))
    x.requires_grad_()
    f = lambda t: L.dropout(t, 0.5, state(3))  # noqa: E731  (scale 2: all products and sums below are exact)
    f(x).backward(g)
    assert (f(x + d) - f(x - d)).mul(g).sum() == 2 * (x.grad * d).sum()


@gpu
def test_second_derivative_is_refused(cuda, lib):
    x = torch.randn(10, device="cuda", requires_grad=True)
    y, = torch.autograd.grad(L.dropout(x, 0.5, state(3)).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        y.sum().backward()
