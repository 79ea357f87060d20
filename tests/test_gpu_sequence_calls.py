"""How the sequence operators are called: from several host threads, with forward-mode tangents, with
tensors that autograd watches, in evaluation, on a device that is not the current one."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_norms_from_two_host_threads():
    """Two widths that share a kernel and ask for different amounts of shared memory, launched from two
    threads on two streams: no launch fails and each has the bits it has alone."""
    import ctypes
    from delrec import _lib
    from delrec.block_norm import block_join
    fn = _lib.lib().delrec_block_norm_forward
    failed, wrong, start = [], [], threading.Barrier(2)

    def go(N):
        T, B, stream = 4, 3, torch.cuda.Stream()
        x, y, u = (torch.randn(T, B, N, device="cuda") for _ in range(3))
        want = block_join(x, y, gate=u, next_norm=True)
        out, n = torch.empty_like(x), torch.empty_like(x)
        block = _lib.Block(T, B, N, 0, 1, 0, 1e-5, 0, *(B * N, N) * 5)
        args = (ctypes.byref(block), x.data_ptr(), y.data_ptr(), u.data_ptr(), None, None, None, None, out.data_ptr(),
                n.data_ptr(), None, None, stream.cuda_stream)
        torch.cuda.synchronize()
        start.wait()
        failed.append(sum(fn(*args) != 0 for _ in range(20000)))     # ctypes lets the other thread in
        stream.synchronize()
        if not (torch.equal(out, want[0]) and torch.equal(n, want[1])):
            wrong.append(N)

    threads = [threading.Thread(target=go, args=(N,)) for N in (2048, 1920)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert failed == [0, 0] and not wrong


def test_forward_mode_derivatives_are_refused():
    """A dual tensor needs no gradient of its own; its tangent is not dropped without a word."""
    import torch.autograd.forward_ad as fw
    from delrec.block_norm import block_join, block_norm
    from delrec.gated import gated_scan, gated_step
    z, f, h0, w = (torch.randn(s, device="cuda") for s in ((5, 2, 8), (5, 2, 8), (2, 8), (8,)))
    with fw.dual_level():
        dz, dh, dw = (fw.make_dual(t, torch.ones_like(t)) for t in (z, h0, w))
        for call in (lambda: gated_scan(dz, f), lambda: gated_scan(z, dz), lambda: gated_scan(z, f, dh),
                     lambda: gated_step(dz[0], f[0]), lambda: gated_step(z[0], dz[0]),
                     lambda: gated_step(z[0], f[0], dh), lambda: block_norm(dz), lambda: block_norm(z, dw),
                     lambda: block_join(z, dz), lambda: block_join(z, f, gate=dz), lambda: block_join(z, f, dw),
                     lambda: block_join(z, f, scale=dw), lambda: block_join(z, f, next_weight=dw)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    call()
        want = gated_scan(z, f, h0)
    # outside the level, and inside it without a tangent, the calls run
    for a, b in zip(gated_scan(z, f, h0), want):
        assert torch.equal(a, b)


def test_a_state_updated_in_place_is_seen_by_autograd():
    from delrec.gated import gated_step
    z, f, state = (torch.randn(2, 8, device="cuda") for _ in range(3))
    w = torch.randn(2, 8, device="cuda", requires_grad=True)
    saved = (state * w).sum()             # keeps state for w's gradient
    gated_step(z, f, state, out=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    with pytest.raises(RuntimeError, match="out"):
        gated_step(z, f, state, out=torch.zeros(2, 8, device="cuda", requires_grad=True))
    with torch.inference_mode():          # a streaming state has no version there
        s = torch.zeros(2, 8, device="cuda")
        h, _ = gated_step(z, f, s, out=s)
    assert torch.equal(h, s)


@pytest.mark.parametrize("guard", [torch.no_grad, torch.inference_mode])
def test_evaluation_keeps_nothing_in_8_bits(guard, monkeypatch):
    """Without gradients a checkpoint8 layer is the plain one: nothing is packed, and the sums have the
    plain order."""
    from delrec import linear
    plain = linear.Linear(700, 130, binary_input=False).cuda()
    keep = linear.Linear(700, 130, binary_input=False, checkpoint8=True).cuda()
    keep.load_state_dict(plain.state_dict())
    x = torch.randn(300, 700, device="cuda")
    monkeypatch.setattr(linear, "empty8", lambda *a: pytest.fail("packed in evaluation"))
    with guard():
        assert torch.equal(keep(x), plain(x))
        assert torch.equal(linear.linear(x, keep.weight, keep.bias, binary_input=False, checkpoint8=True), plain(x))


def test_evaluation_of_two_graphs_with_8_bit_projections(monkeypatch):
    """Captured evaluation passes of checkpoint8 layers share no scratch: replayed on two streams at once."""
    from delrec import _lib
    from delrec.linear import linear
    monkeypatch.setattr(_lib, "workspace", lambda *a: pytest.fail("scratch that outlives the call"))
    sets = [[torch.randn(s, device="cuda") for s in ((900, 130), (70, 130))] for _ in range(2)]
    for args in sets:
        args[1].requires_grad_(True)

    def go(x, w):
        with torch.no_grad():
            return linear(x, w, binary_input=False, checkpoint8=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [go(*args) for args in sets]
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for args in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(go(*args))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert torch.equal(a, b)


def test_linear8_makes_its_tensors_device_current(monkeypatch):
    """The 8-bit projection launches with its tensors' device current, whichever was."""
    from delrec.linear import linear
    x = torch.randn(20, 40, device="cuda", requires_grad=True)
    w = torch.randn(10, 40, device="cuda", requires_grad=True)

    def go():
        out = linear(x, w, checkpoint8=True)
        return (out.detach(), *torch.autograd.grad(out, (x, w), torch.ones_like(out)))

    want = go()
    entered = []
    guard = torch.cuda.device

    class Recorded(guard):
        def __init__(self, device):
            super().__init__(device)
            entered.append(device)

    # another device seems to be current
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    monkeypatch.setattr(torch.cuda, "device", Recorded)
    got = go()
    assert entered == [0, 0, 0]            # the test for spikes, forward, backward
    monkeypatch.undo()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_gates_without_channels_get_zero_gradients():
    """N = 0 with gates: every gate's sum over its channels is empty."""
    from delrec.gated import gated_scan
    z = torch.randn(6, 3, 0, device="cuda", requires_grad=True)
    f = torch.randn(6, 3, 4, device="cuda", requires_grad=True)
    poison = torch.full((6, 3, 4), float("nan"), device="cuda")
    h, hT = gated_scan(z, f)
    del poison
    dz, df = torch.autograd.grad((h, hT), (z, f), (torch.ones_like(h), torch.ones_like(hT)))
    assert dz.shape == z.shape and torch.equal(df, torch.zeros_like(f))
