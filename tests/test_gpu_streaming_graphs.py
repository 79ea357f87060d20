"""Streaming modules captured in a graph: every replay takes the state further."""

import pytest
import torch

pytestmark = pytest.mark.gpu
N, S, B, T = 24, 8, 3, 12


def _modules(kind):
    from delrec.neuron import GatedIntegrator, SelectiveIntegrator, ShortConv
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)   # noqa: E731
    torch.manual_seed(3)
    if kind == "conv":
        return ShortConv(N, 4, step_mode="s").cuda(), (r(T, B, N),)
    if kind == "conv1":
        return ShortConv(N, 1, step_mode="s").cuda(), (r(T, B, N),)
    if kind == "gated":
        return GatedIntegrator(step_mode="s"), (r(T, B, N), r(T, B, N))
    return SelectiveIntegrator(N, S, step_mode="s").cuda(), (r(T, B, N), r(T, B, N), r(T, B, S), r(T, B, S), r(T, B, N))


@pytest.mark.parametrize("kind", ["conv", "conv1", "scan", "gated"])
def test_replays_of_a_captured_step_stream(kind):
    m, seq = _modules(kind)
    with torch.no_grad():
        want = [m(*(v[t] for v in seq)) for t in range(T)]
        last = m.v
        m.reset()
        m(*(v[0] for v in seq))            # the state there is before the capture
        now = [v[1].clone() for v in seq]
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            y = m(*now)
        for t in range(1, T):
            for a, v in zip(now, seq):
                a.copy_(v[t])
            graph.replay()
            assert torch.equal(y, want[t]), t
        assert torch.equal(m.v, last)
        if kind != "conv1":                # starting again
            m.v.zero_()
            for t in range(3):
                for a, v in zip(now, seq):
                    a.copy_(v[t])
                graph.replay()
                assert torch.equal(y, want[t]), t


@pytest.mark.parametrize("kind", ["conv", "scan", "gated"])
def test_a_capture_of_several_steps_and_of_the_first(kind):
    """Three steps in one graph go on from replay to replay; a capture that begins without a state begins anew each time."""
    m, seq = _modules(kind)
    with torch.no_grad():
        want = [m(*(v[t] for v in seq)) for t in range(T)]
        for start in (None, 0):
            m.reset()
            if start is not None:
                m(*(v[0] for v in seq))
            n0 = 0 if start is None else 1
            now = [v[n0:n0 + 3].clone() for v in seq]
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                ys = [m(*(v[k] for v in now)) for k in range(3)]
            for r in range(3):
                at = n0 + (3 * r if start is not None else 0)
                for a, v in zip(now, seq):
                    a.copy_(v[at:at + 3])
                graph.replay()
                for k in range(3):
                    assert torch.equal(ys[k], want[at + k]), (start, r, k)


@pytest.mark.parametrize("kind", ["conv", "scan", "gated"])
def test_an_eager_step_leaves_the_state_before_it(kind):
    """Who keeps a state can go back to it."""
    m, seq = _modules(kind)
    with torch.no_grad():
        for t in range(3):
            m(*(v[t] for v in seq))
        kept, copy = m.v, m.v.clone()
        one = m(*(v[3] for v in seq))
        assert m.v is not kept and torch.equal(kept, copy)
        m.v = kept
        assert torch.equal(m(*(v[3] for v in seq)), one)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("kind", ["conv", "scan", "gated"])
def test_replays_of_a_captured_piece_go_on(kind, train):
    """Pieces of a sequence with ``keep_state``, also with a backward pass in the graph."""
    m, seq = _modules(kind)
    m.step_mode, m.keep_state = "m", True

    def go(piece):
        piece = [v.detach().requires_grad_(train) for v in piece]
        y = m(*piece)
        return [y.detach()] + (list(torch.autograd.grad(y, piece, torch.ones_like(y))) if train else [])

    with torch.set_grad_enabled(train):
        want = [[v.clone() for v in go([v[a:a + 3] for v in seq])] for a in range(0, T, 3)]
        last = m.v.clone()
        m.reset()
        go([v[:3] for v in seq])
        now = [v[3:6].clone() for v in seq]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            kept = m.v
            go(now)                        # before a capture, on another stream, without moving the state
            m.v = kept
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = go(now)
        for k in range(1, T // 3):
            for a, v in zip(now, seq):
                a.copy_(v[3 * k:3 * k + 3])
            graph.replay()
            for a, b in zip(out, want[k]):
                assert torch.equal(a, b), k
        assert torch.equal(m.v, last)


@pytest.mark.parametrize("kind", ["conv", "scan", "gated"])
def test_a_captured_state_outlives_a_reset(kind):
    """Replays go on writing to the state of the capture: no one else is given its memory."""
    m, seq = _modules(kind)
    with torch.no_grad():
        m(*(v[0] for v in seq))
        size, dtype = m.v.numel() * m.v.element_size(), torch.uint8
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            y = m(*(v[1] for v in seq))
        graph.replay()
        torch.cuda.synchronize()
        m.reset()
        m(*(v[0] for v in seq))            # and a state of its own behind a call
        m.reset()
        others = [torch.full((size,), 77, dtype=dtype, device="cuda") for _ in range(64)]
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert all((v == 77).all() for v in others) and torch.isfinite(y).all()
