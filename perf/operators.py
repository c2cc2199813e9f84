"""The operators between two layers of a net, as a user has them run: group norm with an activation, its interval
form, and dropout from a counter-based generator.

`listed()` names the cases, `draw(rng)` gives further ones of the same ranges, `prepare(case, seed)` builds what a
program holds before the call, `run(state)` is one pass, `work(case)` what the pass cannot do without and
`exact(case, seed)` the same results from the definition in 64 bits.  Where `own` is false, `run` computes with
elementary torch operations; where it is true, it makes the calls of the package.

Kinds of case:
  norm     group_norm, channels last: the forward, or with `train` the forward and all its gradients
  bound    group_norm_bound: lower / upper bounds of a box, with `train` the gradients as well
  dropout  dropout of one tensor or of a (value, lower, upper) triple, with `train` the gradients as well
"""
import math

import torch

own = False


def listed():
    return [
        # The head of the '++' nets in training: hidden activations of one batch, all launches and latency.
        {"name": "drop_head_triple", "kind": "dropout", "batch": 512, "channels": 512, "side": 1, "type": "float32", "rate": 0.1, "triple": True, "train": True},
        # Feature maps of somebody's own net: no size is a multiple of anything.
        {"name": "drop_ragged", "kind": "dropout", "batch": 203, "channels": 1333, "side": 5, "type": "float16", "rate": 0.25, "triple": False, "train": True},
        # Feature maps of a large image batch in mixed precision: bandwidth is all there is.
        {"name": "drop_maps", "kind": "dropout", "batch": 64, "channels": 256, "side": 64, "type": "bfloat16", "rate": 0.1, "triple": False, "train": True},
        # One image through a small trained net: the smallest call.
        {"name": "norm_one_image", "kind": "norm", "batch": 1, "channels": 64, "side": 16, "groups": 8, "type": "float32", "act": "relu", "rate": 0.0, "train": False},
        # Evaluation of dense hidden layers, 512 samples: one position per sample.
        {"name": "norm_dense", "kind": "norm", "batch": 512, "channels": 5120, "side": 1, "groups": 32, "type": "float32", "act": "tanh", "rate": 0.0, "train": False},
        # Inference on large feature maps in mixed precision, groups of ten channels.
        {"name": "norm_maps", "kind": "norm", "batch": 32, "channels": 320, "side": 64, "groups": 32, "type": "bfloat16", "act": "silu", "rate": 0.0, "train": False},
        # Training behind a 3 x 3 convolution of distance neurons: 64 feature maps of 16 x 16.
        {"name": "norm_conv_train", "kind": "norm", "batch": 64, "channels": 128, "side": 16, "groups": 32, "type": "float32", "act": "tanh", "rate": 0.0, "train": True},
        # Training on odd sizes with groups that no wide load divides.
        {"name": "norm_ragged_train", "kind": "norm", "batch": 13, "channels": 75, "side": 37, "groups": 5, "type": "float16", "act": "silu", "rate": 0.2, "train": True},
        # Training on maps so large that no sample stays on the chip, with dropout behind the activation.
        {"name": "norm_maps_train", "kind": "norm", "batch": 16, "channels": 128, "side": 160, "groups": 32, "type": "bfloat16", "act": "silu", "rate": 0.1, "train": True},
        # Training of the head on worst-case margins: the box of the feature output, 512 samples.
        {"name": "bound_head_train", "kind": "bound", "batch": 512, "channels": 512, "side": 1, "groups": 16, "act": "tanh", "eps": 8 / 255, "train": True},
        # Certification behind a convolution of distance neurons.
        {"name": "bound_conv", "kind": "bound", "batch": 64, "channels": 128, "side": 16, "groups": 8, "act": "relu", "eps": 8 / 255, "train": False},
        # Certification of a batch of large images.
        {"name": "bound_maps", "kind": "bound", "batch": 32, "channels": 192, "side": 56, "groups": 6, "act": "relu", "eps": 1 / 255, "train": False},
    ]


MOST_BYTES = 100_000_000          # of one direction's inputs in a drawn case


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _shape(rng, most):
    """(batch, groups, channels, side): dense activations or feature maps, half of the channel counts as most people choose them."""
    while True:
        side = 1 if rng.random() < 0.3 else _log(rng, 3, 160)
        batch = _log(rng, 1, 2048 if side == 1 else 64)
        groups = rng.choice([1, 2, 4, 8, 16, 32, 32, rng.randint(1, 24)])
        per = _log(rng, 2, max(4, (5120 if side == 1 else 640) // groups))
        if rng.random() < 0.5:
            per = max(2, per // 8 * 8)
        if batch * groups * per * side * side <= most and groups * per * side * side >= 64:
            return batch, groups, groups * per, side


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm", "bound", "dropout", "dropout"])
    if kind == "dropout":
        triple = rng.random() < 0.3
        kept = "float32" if triple else rng.choice(["float32", "bfloat16", "float16"])
        batch, _, channels, side = _shape(rng, MOST_BYTES // (12 if triple else 4 if kept == "float32" else 2))
        return {"kind": kind, "batch": batch, "channels": channels, "side": side, "type": kept,
                "rate": rng.choice([0.05, 0.1, 0.25, 0.5, round(rng.uniform(0.01, 0.9), 3)]), "triple": triple, "train": rng.random() < 0.7}
    train = rng.random() < 0.6
    kept = rng.choice(["float32", "float32", "bfloat16", "float16"])
    batch, groups, channels, side = _shape(rng, MOST_BYTES // (8 if kind == "bound" else 4 if kept == "float32" else 2))
    case = {"kind": kind, "batch": batch, "channels": channels, "side": side, "groups": groups,
            "act": rng.choice(["identity", "tanh", "silu"] if kind == "norm" else ["identity", "tanh"]) if train else rng.choice(["identity", "relu", "tanh", "silu"]), "train": train}
    if kind == "bound":
        return {**case, "eps": rng.choice([1 / 255, 8 / 255, 0.1])}
    return {**case, "type": kept, "rate": rng.choice([0.0, 0.0, 0.1, 0.3])}


def _maps(gen, case, spread):
    """[batch, channels, side, side] with the channels last in memory, or [batch, channels]."""
    B, C, n = case["batch"], case["channels"], case["side"]
    if n == 1:
        return torch.randn(B, C, generator=gen, device="cuda").mul_(spread)
    return torch.randn(B, n, n, C, generator=gen, device="cuda").mul_(spread).permute(0, 3, 1, 2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    C, train = case["channels"], case["train"]
    kept = getattr(torch, case.get("type", "float32"))
    # what a distance layer gives: positive, far from 0 against its spread, a mean of its own for each channel
    level = 3.0 + 0.5 * torch.randn(C, generator=gen, device="cuda")
    x = _maps(gen, case, 0.5)
    x += level if case["side"] == 1 else level.view(1, C, 1, 1)
    if case["kind"] != "dropout":
        s["weight"] = 1.0 + 0.3 * torch.randn(C, generator=gen, device="cuda")
        s["bias"] = 0.3 * torch.randn(C, generator=gen, device="cuda")
        if train:
            s["weight"].requires_grad_()
            s["bias"].requires_grad_()
    if case["kind"] == "bound" or case.get("triple"):
        # a box around the activations: eps in each direction where it is the input's, wider or narrower behind some layers
        eps = case.get("eps", 0.03)
        wide = torch.rand(x.shape[0], 1, generator=gen, device="cuda") + 0.5
        wide = wide.view(-1, *[1] * (x.dim() - 1))
        s["lower"], s["upper"] = x - eps * wide, x + eps * wide
    if case["kind"] != "bound":
        s["x"] = x.to(kept)
        s["rng"] = torch.tensor([seed * 7919 + 12345678901234567, seed % 1000], dtype=torch.int64, device="cuda")
    names = [n for n in ("x", "lower", "upper") if n in s]
    s["names"] = names
    if train:
        for n in names:
            s[n].requires_grad_()
        s["grads"] = [_maps(gen, case, 1.0).to(s[n].dtype) for n in names]
    return s


# ---- the plain form: elementary operations in 32 bits, in 64 where a sum or a sign asks for them -------------------------


def _threshold(rate):
    """A rate counts in steps of 2^-16."""
    return math.floor(rate * 65536 + 0.5)


def _keep(rng, rate, count, device):
    """Truth values, one for each element by its number: Philox4x32-7 (Salmon, Moraes, Dror and Shaw, 2011) with the counter
    (number / 8, offset) and the seed as key gives eight pieces of 16 bits, the element of number i takes piece i % 8, counted
    from the lowest bits of the first word, and is kept where that piece is at least rate * 2^16."""
    low = 0xFFFFFFFF
    block = torch.arange((count + 7) // 8, dtype=torch.int64, device=device)
    a, b = block & low, block >> 32
    c = (rng[1] & low).expand_as(block)
    d = ((rng[1] >> 32) & low).expand_as(block)
    k0, k1 = rng[0] & low, (rng[0] >> 32) & low
    for _ in range(7):
        p, q = a * 0xD2511F53, c * 0xCD9E8D57           # modulo 2^64: the shifts below take its words apart
        a, b, c, d = ((q >> 32) & low) ^ b ^ k0, q & low, ((p >> 32) & low) ^ d ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    pieces = [t for word in (a, b, c, d) for t in (word & 0xFFFF, word >> 16)]
    return torch.stack(pieces, dim=1).reshape(-1)[:count] >= _threshold(rate)


def _last(t):
    """[batch, channels, ...] -> [batch, positions, channels], the order in which elements are numbered."""
    return t.reshape(t.size(0), t.size(1), -1).transpose(1, 2)


def _first(t, like):
    return t.transpose(1, 2).reshape(like.shape)


def _drop(t, keep, rate):
    return torch.where(keep, t * (65536 / (65536 - _threshold(rate))), torch.zeros((), device=t.device))


def _act(u, act):
    if act == "relu":
        return u.clamp(min=0)
    if act == "tanh":
        return torch.tanh(u)
    return u * torch.sigmoid(u) if act == "silu" else u


def _slope(u, act):
    if act == "relu":
        return (u > 0).to(u.dtype)
    if act == "tanh":
        return 1 - torch.tanh(u) ** 2
    if act == "silu":
        q = torch.sigmoid(u)
        return q * (1 + u * (1 - q))
    return torch.ones_like(u)


def _plain_norm(s):
    x, w, b, G, eps = s["x"].detach(), s["weight"].detach(), s["bias"].detach(), s["groups"], 1e-5
    N, C = x.size(0), x.size(1)
    t = _last(x).float().reshape(N, -1, G, C // G)
    mean = t.mean(dim=(1, 3), keepdim=True)
    t = t - mean
    r = 1.0 / torch.sqrt((t * t).mean(dim=(1, 3), keepdim=True) + eps)
    h = (t * r).reshape(N, -1, C)
    u = h * w + b
    y = _act(u, s["act"])
    keep = _keep(s["rng"], s["rate"], x.numel(), x.device).view(y.shape) if s["rate"] > 0 else None
    if keep is not None:
        y = _drop(y, keep, s["rate"])
    y = _first(y, x).to(x.dtype)
    if not s["train"]:
        return y
    d = _last(s["grads"][0]).float()
    if keep is not None:
        d = _drop(d, keep, s["rate"])
    d = d * _slope(u, s["act"])
    gb, gw = d.sum(dim=(0, 1)), (d * h).sum(dim=(0, 1))
    d = (d * w).view(N, -1, G, C // G)
    h = h.view(d.shape)
    gx = r * (d - d.mean(dim=(1, 3), keepdim=True) - h * (d * h).mean(dim=(1, 3), keepdim=True))
    return [y, _first(gx.reshape(N, -1, C), x).to(x.dtype), gw, gb]


def _plain_bound(s):
    """In 64 bits: which end of an interval a bound takes is decided next to 0."""
    shape, w, b, G, eps = s["lower"].shape, s["weight"].detach().double(), s["bias"].detach().double(), s["groups"], 1e-5
    N, C = shape[0], shape[1]
    lo, up = (_last(s[n].detach()).double().reshape(N, -1, G, C // G) for n in ("lower", "upper"))
    M = lo.size(1) * lo.size(3)
    both = lambda t: t.mean(dim=(1, 3), keepdim=True)  # noqa: E731
    ml, mu = both(lo), both(up)
    c, r = (lo + up) / 2 - (ml + mu) / 2, (up - lo) / 2
    sd, rho = torch.sqrt(both(c * c)), torch.sqrt(both(r * r))
    near = (sd - rho).clamp(min=0)
    tight, wide = 1.0 / torch.sqrt(near * near + eps), 1.0 / torch.sqrt((sd + rho) ** 2 + eps)
    n0, n1 = lo - mu + (up - lo) / M, up - ml - (up - lo) / M
    s0, s1 = torch.where(n0 >= 0, wide, tight), torch.where(n1 >= 0, tight, wide)
    most = math.sqrt(M - 1)
    z0, z1 = (n0 * s0).clamp(min=-most), (n1 * s1).clamp(max=most)
    flat = lambda t: t.reshape(N, -1, C)  # noqa: E731
    swap = w < 0
    v0 = torch.where(swap, flat(z1), flat(z0)) * w + b
    v1 = torch.where(swap, flat(z0), flat(z1)) * w + b
    y0, y1 = _act(v0, s["act"]), _act(v1, s["act"])
    if s["act"] == "silu":                                   # falls to its least value and rises behind it
        least = -1.278464542761074
        inside = (v0 < least) & (v1 > least)
        y0, y1 = torch.where(inside, _act(torch.full_like(y0, least), "silu"), torch.minimum(y0, y1)), torch.maximum(y0, y1)
    y0, y1 = _first(y0, s["lower"]).float(), _first(y1, s["lower"]).float()
    if not s["train"]:
        return [y0, y1]
    g0, g1 = (_last(g).double() * _slope(v, s["act"]) for g, v in zip(s["grads"], (v0, v1)))
    gb = (g0 + g1).sum(dim=(0, 1))
    gw = (g0 * torch.where(swap, flat(z1), flat(z0)) + g1 * torch.where(swap, flat(z0), flat(z1))).sum(dim=(0, 1))
    z_0, z_1 = (torch.where(swap, g1, g0) * w).view(lo.shape), (torch.where(swap, g0, g1) * w).view(lo.shape)
    z_0, z_1 = torch.where(n0 * s0 > -most, z_0, torch.zeros_like(z_0)), torch.where(n1 * s1 < most, z_1, torch.zeros_like(z_1))
    a0, a1 = z_0 * s0, z_1 * s1
    on_wide = both(torch.where(n0 >= 0, z_0 * n0, torch.zeros_like(n0)) + torch.where(n1 >= 0, torch.zeros_like(n1), z_1 * n1)) * wide ** 3 * (sd + rho)
    on_tight = both(torch.where(n0 >= 0, torch.zeros_like(n0), z_0 * n0) + torch.where(n1 >= 0, z_1 * n1, torch.zeros_like(n1))) * tight ** 3 * near
    dc = -(on_wide + on_tight) * c / sd.clamp(min=1e-300)
    dr = (on_tight - on_wide) * r / rho.clamp(min=1e-300)
    gl = a0 * (1 - 1 / M) + a1 / M - both(a1) + (dc - dr) / 2
    gu = a1 * (1 - 1 / M) + a0 / M - both(a0) + (dc + dr) / 2
    return [y0, y1, _first(flat(gl), s["lower"]).float(), _first(flat(gu), s["lower"]).float(), gw.float(), gb.float()]


def _plain_dropout(s):
    keep = None
    outs = []
    for t in [s[n].detach() for n in s["names"]] + s.get("grads", []):
        if keep is None:
            keep = _keep(s["rng"], s["rate"], t.numel(), t.device).view(_last(t).shape)
        outs.append(_first(_drop(_last(t).float(), keep, s["rate"]), t).to(t.dtype))
    return outs


def run(state):
    s = state
    if not own:
        with torch.no_grad():
            return {"norm": _plain_norm, "bound": _plain_bound, "dropout": _plain_dropout}[s["kind"]](s)
    import linfdist_b200 as L
    if s["kind"] == "norm":
        inputs = (s["x"], s["weight"], s["bias"])
        outs = [L.group_norm(s["x"], s["groups"], s["weight"], s["bias"], activation=s["act"], rate=s["rate"], rng=s["rng"] if s["rate"] > 0 else None)]
    elif s["kind"] == "bound":
        inputs = (s["lower"], s["upper"], s["weight"], s["bias"])
        outs = list(L.group_norm_bound(s["lower"], s["upper"], s["groups"], s["weight"], s["bias"], activation=s["act"]))
    else:
        inputs = [s[n] for n in s["names"]]
        outs = L.dropout(s["x"], s["rate"], s["rng"], s.get("lower"), s.get("upper"))
        outs = list(outs) if s["triple"] else [outs]
    if not s["train"]:
        return outs[0] if s["kind"] == "norm" else outs
    return [y.detach() for y in outs] + list(torch.autograd.grad(outs, inputs, s["grads"]))


def work(case):
    n = case["batch"] * case["channels"] * case["side"] ** 2
    size = 4 if case.get("type", "float32") == "float32" else 2
    tensors = 2 if case["kind"] == "bound" else 3 if case.get("triple") else 1
    passes = 4 if case["train"] else 2                  # inputs and outputs, with their gradients
    nbytes = n * size * tensors * passes
    if case["kind"] == "dropout":
        return {"bytes": float(nbytes), "flops": float(n * (passes // 2) * tensors)}
    nbytes += 4 * case["channels"] * passes
    return {"bytes": float(nbytes), "flops": float(n * tensors * (12 if not case["train"] else 36))}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------


def _words(seed, offset, count, device):
    """The generator's pieces of 16 bits, products taken apart into pieces of 16 bits."""
    half, low = 0xFFFF, 0xFFFFFFFF

    def product(x, k):
        x0, x1, k0, k1 = x & half, x >> 16, k & half, k >> 16
        mid = x1 * k0 + ((x0 * k0) >> 16)
        side = x0 * k1 + (mid & half)
        return x1 * k1 + (mid >> 16) + (side >> 16), ((side & half) << 16) | ((x0 * k0) & half)

    i = torch.arange((count + 7) // 8, dtype=torch.int64, device=device)
    v = [i % 2 ** 32, i // 2 ** 32, torch.full_like(i, offset & low), torch.full_like(i, (offset >> 32) & low)]
    key = [seed & low, (seed >> 32) & low]
    for turn in range(7):
        h0, l0 = product(v[0], 0xD2511F53)
        h1, l1 = product(v[2], 0xCD9E8D57)
        v = [h1 ^ v[1] ^ ((key[0] + turn * 0x9E3779B9) & low), l1, h0 ^ v[3] ^ ((key[1] + turn * 0xBB67AE85) & low), l0]
    return torch.stack([t for word in v for t in (word % 65536, word // 65536)], dim=1).view(-1)[:count]


def exact(case, seed):
    s = prepare(case, seed)
    train, kind = case["train"], case["kind"]
    ins = [s[n].detach().double().requires_grad_(train) for n in s["names"]]
    N, C, shape = ins[0].size(0), ins[0].size(1), ins[0].shape
    factor = None
    if case.get("rate", 0) > 0:
        key, offset = s["rng"].tolist()
        words = _words(key, offset, ins[0].numel(), ins[0].device).view(N, -1, C).movedim(2, 1).reshape(shape)
        rate = round(case["rate"] * 65536) / 65536
        factor = (words.double() / 65536 >= rate).double() / (1 - rate)
        del words
    leaves = list(ins)
    if kind == "dropout":
        outs = [t * factor for t in ins]
    else:
        w, b = (s[n].detach().double().requires_grad_(train) for n in ("weight", "bias"))
        leaves += [w, b]
        G = case["groups"]
        as_map = lambda t: t.view(1, C, *[1] * (ins[0].dim() - 2))  # noqa: E731
        f = {"identity": lambda t: t, "relu": torch.relu, "tanh": torch.tanh, "silu": torch.nn.functional.silu}[case["act"]]
        if kind == "norm":
            outs = [f(torch.nn.functional.group_norm(ins[0], G, w, b, eps=1e-5))]
            outs = [outs[0] * factor] if factor is not None else outs
        else:
            lo, up = (t.reshape(N, G, -1) for t in ins)
            M = lo.size(2)
            centre, radius = (lo + up) / 2, (up - lo) / 2
            sd = centre.var(dim=2, unbiased=False, keepdim=True).clamp(min=1e-300).sqrt()
            rho = radius.square().mean(dim=2, keepdim=True).sqrt()
            ends = [((sd + rho).square() + 1e-5).rsqrt(), (torch.relu(sd - rho).square() + 1e-5).rsqrt()]
            rest_lo, rest_up = lo.sum(2, keepdim=True) - lo, up.sum(2, keepdim=True) - up
            least, most = (lo * (M - 1) - rest_up) / M, (up * (M - 1) - rest_lo) / M
            z = [torch.minimum(least * ends[0], least * ends[1]).clamp(min=-math.sqrt(M - 1)),
                 torch.maximum(most * ends[0], most * ends[1]).clamp(max=math.sqrt(M - 1))]
            z = [t.reshape(shape) * as_map(w) + as_map(b) for t in z]
            turned = (as_map(w) < 0).expand(shape)
            v0, v1 = torch.where(turned, z[1], z[0]), torch.where(turned, z[0], z[1])
            if case["act"] == "silu":
                bottom = torch.full_like(v0, -1.278464542761074)
                outs = [torch.where((v0 < bottom) & (v1 > bottom), f(bottom), torch.minimum(f(v0), f(v1))), torch.maximum(f(v0), f(v1))]
            else:
                outs = [f(v0), f(v1)]
    got = [y.detach() for y in outs]
    if train:
        got += list(torch.autograd.grad(outs, leaves, [g.double() for g in s["grads"]]))
    return got[0] if kind == "norm" and not train else got
