"""Group norm and dropout called in ways of their own: from several threads at once, traced, under transforms and checkpoints, by replicas."""
import threading

import pytest
import torch

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
