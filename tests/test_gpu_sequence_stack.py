"""The sequence operators together: a two-block gated network on a padded batch, trained for a
step, streamed step by step, and captured in a graph."""

import pytest
import torch

from oracle import sequence_oracle as O

pytestmark = pytest.mark.gpu

T, B, N, G = 40, 3, 48, 48


class Stack(torch.nn.Module):
    """Per block: norm -> projections (z, f, gate) -> gated integrator -> join with the next norm."""

    def __init__(self, checkpoint8=False):
        super().__init__()
        from delrec.linear import Linear
        from delrec.neuron import BlockJoin, BlockNorm, GatedIntegrator
        self.first = BlockNorm(N)
        self.proj = torch.nn.ModuleList(Linear(N, 3 * N, binary_input=False, checkpoint8=checkpoint8)
                                        for _ in range(2))
        self.core = torch.nn.ModuleList(GatedIntegrator(checkpoint8=checkpoint8) for _ in range(2))
        self.join = torch.nn.ModuleList(BlockJoin(N, "silu", 0.5, next_norm=i == 0) for i in range(2))

    def forward(self, x, lengths=None):
        n = self.first(x, lengths)
        for proj, core, join in zip(self.proj, self.core, self.join):
            z, f, u = proj(n).split(N, -1)
            h = core(z, f, lengths) if lengths is not None else core(z, f)
            r = join(x, h, u, lengths)
            x, n = r if isinstance(r, tuple) else (r, None)
        return x


def _reference(params, x, lengths):
    """The same network in float64 with autograd, on the CPU."""
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in params.items()}
    live = (torch.arange(T)[:, None] < lengths[None, :])[..., None]
    x = x.detach().double().cpu().requires_grad_(True)
    s = torch.where(live, x, torch.zeros_like(x))
    _, n = O.block_join(s, None, None, None, "none", None, p["first.weight"], 1e-5, True)
    for i in range(2):
        z, f, u = (n @ p[f"proj.{i}.weight"].t() + p[f"proj.{i}.bias"]).split(N, -1)
        h, hs = torch.zeros(B, N, dtype=torch.float64), []
        for t in range(T):
            a = torch.sigmoid(f[t])
            h = torch.where(live[t], a * h + (1 - a) * z[t], h)
            hs.append(torch.where(live[t], h, torch.zeros_like(h)))
        nw = p.get(f"join.{i}.next_weight")
        s, n = O.block_join(s, torch.stack(hs), p[f"join.{i}.weight"], u, "silu", p[f"join.{i}.scale"], nw, 1e-5,
                            nw is not None)
        s = torch.where(live, s, torch.zeros_like(s))
    return s, p, x


def _case():
    torch.manual_seed(3)
    model = Stack().cuda()
    x = torch.randn(T, B, N, device="cuda")
    g = torch.randn(T, B, N, device="cuda")
    return model, x, g, torch.tensor([T, 17, 1])


def test_training_pass():
    """Outputs and every gradient against float64.  Relative to each tensor's largest entry:
    fp32 projections to 1e-5 (their own tests' tolerance), three in a row on the longest path
    and as many again backward, so 1e-4."""
    model, x, g, lengths = _case()
    x.requires_grad_(True)
    out = model(x, lengths.cuda())
    params = dict(model.named_parameters())
    grads = torch.autograd.grad(out, [x, *params.values()], g)
    ref, p, xr = _reference(params, x, lengths)
    want = torch.autograd.grad(ref, [xr, *p.values()], g.double().cpu())
    for got, w, name in zip((out.detach(), *grads), (ref.detach(), *want), ("out", "x", *params)):
        err = (got.double().cpu() - w).abs().max() / w.abs().max()
        assert err < 1e-4, f"{name}: {err:.2e}"


def test_checkpoints_keep_the_forward_and_come_near_the_gradients():
    """8-bit checkpoints: the same output to fp32 accuracy; the gradients point the same way.  Each restored value
    is within 2^-7 of its group's largest, so a gradient summed over T B positions of random
    sign stays within a few percent of its norm."""
    model, x, g, lengths = _case()
    small = Stack(checkpoint8=True).cuda()
    small.load_state_dict(model.state_dict())
    a, b = model(x, lengths.cuda()), small(x, lengths.cuda())
    assert (a - b).abs().max() <= 1e-4 * a.abs().max()
    ga = torch.autograd.grad(a, list(model.parameters()), g)
    gb = torch.autograd.grad(b, list(small.parameters()), g)
    for u, v in zip(ga, gb):
        assert (u - v).norm() <= 0.05 * u.norm()


def test_streaming_is_the_whole_sequence():
    from delrec.utils import reset_states
    model, x, _, _ = _case()
    with torch.no_grad():
        whole = model(x)
        for core in model.core:
            core.step_mode = "s"
        for _ in range(2):
            reset_states(model)
            for t in range(T):
                h = x[t:t + 1]
                n = model.first(h)
                for proj, core, join in zip(model.proj, model.core, model.join):
                    z, f, u = proj(n).split(N, -1)
                    r = join(h, core(z[0], f[0])[None], u)
                    h, n = r if isinstance(r, tuple) else (r, None)
                torch.testing.assert_close(h[0], whole[t], rtol=1e-4, atol=1e-4)


def test_pieces_with_kept_state():
    """A long sequence in pieces of odd lengths, the state kept between them."""
    from delrec.neuron import GatedIntegrator
    from delrec.utils import reset_states
    torch.manual_seed(1)
    z, f = torch.randn(T, B, N, device="cuda"), torch.randn(T, B, 8, device="cuda")
    whole = GatedIntegrator()(z, f)
    m = GatedIntegrator(keep_state=True)
    for _ in range(2):
        got = torch.cat([m(z[a:b], f[a:b]) for a, b in ((0, 1), (1, 18), (18, 40))])
        torch.testing.assert_close(got, whole, rtol=2 ** -18, atol=2 ** -18)
        reset_states(m)


def test_captured_training_pass():
    model, x, g, lengths = _case()
    lengths = lengths.cuda()
    params = list(model.parameters())

    def go():
        out = model(x, lengths)
        return (out.detach(), *torch.autograd.grad(out, params, g))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        go()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = go()
    x.copy_(torch.randn_like(x))
    lengths.copy_(torch.tensor([5, T, 0]))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, go()):
        assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements (4.3 GB each): the last rows are those of a call on them alone."""
    from delrec.block_norm import block_norm
    from delrec.checkpoint8 import pack8, unpack8
    from delrec.gated import gated_scan
    Tb, Bb, Nb = 70000, 60, 520
    z = torch.empty(Tb, Bb, Nb, dtype=torch.bfloat16, device="cuda").normal_()
    assert z.numel() > 2 ** 31
    f = torch.full((1, 1, 1), 3.0, dtype=torch.bfloat16, device="cuda").expand(Tb, Bb, 1)
    tol = dict(rtol=2.0 ** -7, atol=2.0 ** -10.5)      # a step of bf16, sums in another order
    h, hT = gated_scan(z, f)
    one, last = gated_scan(z[:, -1:].contiguous(), f[:, -1:])
    torch.testing.assert_close(h[:, -1:], one, **tol)
    torch.testing.assert_close(hT[-1:], last, rtol=0, atol=2.0 ** -10.5)
    del h
    n = block_norm(z)
    torch.testing.assert_close(n[-3:], block_norm(z[-3:].clone()), rtol=2.0 ** -7, atol=2.0 ** -18)
    del n
    p = pack8(z)
    assert torch.equal(unpack8(p._replace(q=p.q[-3:], e=p.e[-3:])), unpack8(pack8(z[-3:].clone())))
    assert torch.equal(unpack8(p)[-3:], unpack8(pack8(z[-3:].clone())))


def test_backward_past_32_bits():
    from delrec.gated import gated_scan
    Tb, Bb, Nb = 4200, 1024, 512
    z = torch.empty(Tb, Bb, Nb, dtype=torch.bfloat16, device="cuda").normal_()
    f = torch.full((1, 1, 1), 1.0, dtype=torch.bfloat16, device="cuda").expand(Tb, Bb, Nb)
    g = torch.ones(1, 1, 1, dtype=torch.bfloat16, device="cuda").expand(Tb, Bb, Nb)
    for keep in (False, True):
        zz = z.detach().requires_grad_(True)
        h, _ = gated_scan(zz, f, checkpoint8=keep)
        (dz,) = torch.autograd.grad(h, zz, g)
        zs = z[:, -1:].clone().requires_grad_(True)
        hs, _ = gated_scan(zs, f[:, -1:], checkpoint8=keep)
        (ds,) = torch.autograd.grad(hs, zs, g[:, -1:])
        torch.testing.assert_close(h[:, -1:], hs, rtol=2.0 ** -7, atol=2.0 ** -10.5)
        torch.testing.assert_close(dz[:, -1:], ds, rtol=2.0 ** -7, atol=2.0 ** -10.5)
        del h, dz


def test_second_derivatives_are_refused():
    from delrec.block_norm import block_norm
    from delrec.gated import gated_scan
    x = torch.randn(5, 2, 8, device="cuda", requires_grad=True)
    for fn in (lambda: gated_scan(x, x)[0], lambda: block_norm(x)):
        out = fn()
        go = torch.randn_like(out).requires_grad_(True)
        (g,) = torch.autograd.grad(out, x, go, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


def test_two_streams_at_once():
    """Training passes of two models' operators on two streams, interleaved: each has the results it has
    alone."""
    model, x, g, lengths = _case()
    lengths = lengths.cuda()
    small = Stack(checkpoint8=True).cuda()
    small.load_state_dict(model.state_dict())

    def go(m):
        out = m(x, lengths)
        return (out.detach(), *torch.autograd.grad(out, list(m.parameters()), g))

    want = [go(model), go(small)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, m in enumerate((model, small)):
            with torch.cuda.stream(streams[i]):
                got[i].append(go(m))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(a, b)


def test_two_graphs_with_8_bit_projections_at_once():
    """Captured training passes with 8-bit projections share no scratch: replayed on two streams at once."""
    from delrec.linear import linear
    gen = torch.Generator(device="cuda").manual_seed(4)
    sets = [[torch.randn(s, device="cuda", generator=gen) for s in ((900, 130), (70, 130), (900, 70))] for _ in range(2)]

    def go(x, w, g):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        out = linear(x, w, binary_input=False, checkpoint8=True)
        return (out.detach(), *torch.autograd.grad(out, (x, w), g))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        go(*sets[0])
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for args in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(go(*args))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for st, graph in zip(streams, graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for got, args in zip(outs, sets):
        for a, b in zip(got, go(*args)):
            assert torch.equal(a, b)
