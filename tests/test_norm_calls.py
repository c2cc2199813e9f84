"""Group norm and dropout called in ways of their own: from several threads at once, traced, under transforms and checkpoints, by replicas."""
import os
import pickle
import sys
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import linfdist_b200 as L

gpu = pytest.mark.gpu


@gpu
def test_two_threads_with_two_sizes(cuda, lib):
    """The same kernel with 51 and 64 KB of shared memory for each CTA from two threads at once: no call sees the other's limit.  The library's
    own entry point, call after call, so that the threads are inside it at the same time."""
    wrong = []
    begin = threading.Barrier(2)
    data = [torch.randn(8, n, 16, device="cuda") for n in (1000, 800)]
    want = [L.group_norm(x.movedim(-1, 1), 1).movedim(1, -1) for x in data]
    assert all(lib.linf_group_norm_workspace_bytes(8, 16, 1, x.size(1), 0, 0) == 0 for x in data)        # kept: one launch
    torch.cuda.synchronize()

    def work(k):
        x, y, n = data[k], torch.empty_like(data[k]), data[k].size(1)
        stream = torch.cuda.Stream()
        args = (x.data_ptr(), None, None, 8, 16, 1, n, 0, 0, 1e-5, 0, 0.0, None, y.data_ptr(), None, None, None, 0, stream.cuda_stream)
        begin.wait()
        codes = [lib.linf_group_norm_forward(*args) for _ in range(6000)]
        stream.synchronize()
        if any(codes) or not torch.equal(y, want[k]):
            wrong.append(f"thread {k}: {sum(c != 0 for c in codes)} calls refused")

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_forward_mode_tangent_counts_as_a_gradient():
    """What a call without gradients would lose."""
    import torch.autograd.forward_ad as fw
    wants = L.group_norm.__globals__["_wants_grad"]
    x, w = torch.randn(2, 8), torch.ones(8)
    assert not wants(x, w, None) and wants(x, w.clone().requires_grad_())
    with fw.dual_level():
        assert not wants(x, w) and wants(fw.make_dual(x, x), w) and wants(x, None, fw.make_dual(w, w))
        with torch.no_grad():
            assert wants(fw.make_dual(x, x), w)
    seen = []
    torch.func.jvp(lambda t: (seen.append(wants(t)), t)[1], (x,), (x,))
    assert seen == [True]


@gpu
@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_mode_derivatives_are_refused(cuda, lib, which):
    """A tangent of the input, the weight or the bias: an error and not a result without one."""
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        a = [torch.randn(2, 8, device="cuda"), torch.ones(8, device="cuda"), torch.zeros(8, device="cuda")]
        a[which] = fw.make_dual(a[which], torch.ones_like(a[which]))
        for call in (lambda: L.group_norm(a[0], 2, a[1], a[2]), lambda: L.group_norm_bound(a[0], a[0], 2, a[1], a[2])):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
    x = torch.randn(2, 8, device="cuda")
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda t: L.group_norm(t, 2), (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: L.group_norm(t, 2))(x.view(2, 1, 8))


def test_tracing_is_refused():
    """A traced call would give the memory of its result and nothing in it."""
    x, rng = torch.randn(2, 8), torch.zeros(2, dtype=torch.int64)
    for call in (lambda t: L.group_norm(t, 2), lambda t: L.group_norm_bound(t, t, 2)[0], lambda t: L.BoundGroupNorm(2, 8)(t)[0],
                 lambda t: t * L.dropout_next(rng)[0]):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, x)


class _ByHand(torch.autograd.Function):
    """Dropout on the CPU: elements whose number has the parity of the offset are kept."""

    @staticmethod
    def forward(ctx, x, rate, used):
        ctx.keep = (torch.arange(x.numel()).view(x.shape) + int(used[1])) % 2 == 0
        return x * ctx.keep

    @staticmethod
    def backward(ctx, g):
        return g * ctx.keep, None, None


@pytest.fixture
def by_hand(monkeypatch):
    """The modules of this package with the library's two calls done on the CPU."""
    module = sys.modules[L.BoundDropout.__module__]

    def draw(state, replica):
        used = state.clone()
        used[0] += replica
        state[1] += 1
        return used
    monkeypatch.setattr(module, "_draw", draw)
    monkeypatch.setattr(module, "dropout", _ByHand.apply)


@pytest.mark.parametrize("nested", [False, True])
def test_checkpoints_get_the_masks_of_the_first_run(by_hand, nested):
    """Value and gradient have the same mask, twice in a row and with checkpoints of several calls; the offset counts the first runs alone."""
    drop, other = L.BoundDropout(0.5, seed=1).train(), L.BoundDropout(0.5, seed=2).train()
    keep = dict(use_reentrant=False, context_fn=L.checkpoint_masks)

    def block(t):
        t = checkpoint(lambda s: drop(s * 2)[0], t, **keep) if nested else drop(t * 2)[0]
        return other(drop(torch.cat([t, t]).exp())[0])[0]

    x = torch.rand(12, requires_grad=True)
    ys = [checkpoint(block, x, **keep) for _ in range(3)]                     # all before the first backward pass
    assert drop.rng[1] == 6 and other.rng[1] == 3
    got = [torch.autograd.grad(y.sum(), x, retain_graph=True)[0] for y in ys]
    again = [torch.autograd.grad(y.sum(), x)[0] for y in reversed(ys)]
    assert drop.rng[1] == 6 and other.rng[1] == 3
    drop.rng[1], other.rng[1] = 0, 0
    for y, g, h in zip(ys, got, reversed(again)):
        want = block(x) if not nested else None
        if want is not None:
            assert torch.equal(y, want) and torch.equal(g, torch.autograd.grad(want.sum(), x)[0])
        assert torch.equal(g, h) and ((g != 0) <= (y.view(2, 12) != 0).any(0)).all()


def test_checkpoints_without_the_masks_are_refused(by_hand):
    drop = L.BoundDropout(0.5, seed=1).train()
    x = torch.rand(12, requires_grad=True)
    for kw in (dict(use_reentrant=False), dict(use_reentrant=True)):
        y = checkpoint(lambda t: drop(t * 2)[0].exp(), x, **kw)
        with pytest.raises(RuntimeError, match="checkpoint_masks"):
            y.sum().backward()
    count = [0]

    def changes(t):
        count[0] += 1
        return drop(drop(t)[0] if count[0] > 1 else t)[0].exp()
    y = checkpoint(changes, x, use_reentrant=False, context_fn=L.checkpoint_masks)
    with pytest.raises(RuntimeError, match="other masks|different number"):
        y.sum().backward()
    assert not sys.modules[L.BoundDropout.__module__]._masks_of.stack


@gpu
def test_checkpoint_of_norm_and_dropout(cuda, lib):
    """The modules themselves: values and gradients of a checkpointed block are those of the block."""
    norm = L.BoundGroupNorm(4, 32, activation="tanh", dropout=0.25, seed=5).cuda().train()
    drop = L.BoundDropout(0.5, seed=6).cuda().train()
    x = torch.randn(20, 32, device="cuda", requires_grad=True)

    def block(t):
        return [s.sin() for s in drop(*norm(t, t - 0.1, t + 0.1))]

    results = []
    for run in (block, lambda t: checkpoint(block, t, use_reentrant=False, context_fn=L.checkpoint_masks)):
        norm.rng[1] = drop.rng[1] = 0
        ys = run(x)
        results.append([*ys, *torch.autograd.grad(sum(k * y.sum() for k, y in enumerate(ys, 1)), [x, norm.weight, norm.bias])])
        assert norm.rng[1] == 1 and drop.rng[1] == 1
    assert all(torch.equal(a, e) for a, e in zip(*results))


def _replica(rank, world, port, out):
    import torch.distributed as dist
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    from linfdist_b200.train_step import DataParallelStep
    seen = []
    for groups in (None, 4):
        torch.manual_seed(7)                                  # the same net on every rank
        net = torch.nn.Sequential(L.Predictor(8, 16, 3, groups=groups, dropout=0.25))
        step = DataParallelStep(net, L.AdamW(net, lr=0.1))
        module = net[0].drop if groups is None else net[0].norm
        net.load_state_dict(net.state_dict())
        seen.append((module.replica, module.rng.tolist()))
        step.close()
    all_seen = [None] * world
    dist.all_gather_object(all_seen, seen)
    if rank == 0:
        out.put(all_seen)
    dist.destroy_process_group()


def test_replicas_are_numbered():
    """Two CPU ranks with the same net: equal states, which may be loaded and broadcast, and a number of its own for each rank."""
    import torch.multiprocessing as mp
    ctx = mp.get_context("spawn")
    out = ctx.Queue()
    port = 29950 + os.getpid() % 400
    ranks = [ctx.Process(target=_replica, args=(r, 2, port, out)) for r in range(2)]
    for p in ranks:
        p.start()
    seen = out.get(timeout=240)
    for p in ranks:
        p.join(timeout=60)
        assert p.exitcode == 0
    for a, b in zip(*seen):
        assert (a[0], b[0]) == (0, 1) and a[1] == b[1]


def test_seeds_of_the_head():
    for groups in (None, 4):
        heads = [L.Predictor(8, 16, 3, groups=groups, dropout=0.25, seed=s) for s in (3, 4)]
        assert [(h.norm if groups else h.drop).rng.tolist() for h in heads] == [[3, 0], [4, 0]]


@gpu
def test_masks_of_replicas(cuda, lib):
    """Equal states, a seed of its own for each replica; that of replica 0 as it is; the modules' masks differ."""
    rng = [torch.tensor([-5, 40], dtype=torch.int64, device="cuda") for _ in range(3)]
    used = [L.dropout_next(s, replica=k).tolist() for k, s in enumerate(rng)]
    want = [(-5 + k * 0x9E3779B97F4A7C15 + 2 ** 63) % 2 ** 64 - 2 ** 63 for k in range(3)]
    assert used == [[w, 40] for w in want] and all(s.tolist() == [-5, 41] for s in rng)
    x = torch.ones(4, 64, device="cuda")
    for make in (lambda: L.BoundDropout(0.5, seed=1), lambda: L.BoundGroupNorm(4, 64, dropout=0.5, seed=1)):
        masks = []
        for k in (0, 1, 0):
            m = make().cuda().train()
            m.replica = k
            masks.append(m(x + torch.arange(64, device="cuda"))[0] != 0)
        assert torch.equal(masks[0], masks[2]) and not torch.equal(masks[0], masks[1])


def test_what_is_kept_of_sizes_has_an_end(lib, monkeypatch):
    """One entry for each size, up to some thousand."""
    G = sys.modules[L.BoundGroupNorm.__module__]
    monkeypatch.setattr(G, "_scratch", lambda device, need: need)
    device = torch.device("cuda:0")
    for n in range(1, 9001):
        assert G._work_space("linf_group_norm_workspace_bytes", device, n, 8, 2, 1, 0, 1)[1] > 0
    assert len(G._workspace_bytes) <= 4096


def test_nets_saved_whole_before_there_were_norms():
    """A pickled head and a pickled convolution without the newer attributes are what they were."""
    head, conv = L.Predictor(8, 16, 3), L.NormDistConv(4, 32, 3)
    for m, names in ((head, ("groups", "drop")), (conv, ("channels_last",))):
        for name in names:
            del m.__dict__[name]
    head, conv = pickle.loads(pickle.dumps(head)), pickle.loads(pickle.dumps(conv))
    assert conv.channels_last is False
    x, t = torch.randn(5, 8), torch.arange(5) % 3
    y, worst = head(x, x - 0.1, x + 0.1, targets=t)
    triple = head.tanh(*head.fc1(x, x - 0.1, x + 0.1))
    assert all(torch.equal(a, e) for a, e in zip((y, worst), head.fc2(*triple, targets=t)))
    new = pickle.loads(pickle.dumps(L.Predictor(8, 16, 3, dropout=0.5)))
    assert new.drop.rate == 0.5 and new.groups is None
