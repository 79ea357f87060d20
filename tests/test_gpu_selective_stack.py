"""The short convolution, the selective scan and the vocabulary losses together: a two-block network
with a loss per position on a padded batch, trained for a step, streamed step by step, captured in
graphs, on two streams; how the operators are called."""

import pytest
import torch

from oracle import sequence_oracle as O

pytestmark = pytest.mark.gpu

T, B, N, S, V = 36, 3, 48, 8, 211


class Stack(torch.nn.Module):
    """Per block: norm -> projections (x, gate, dt, B, C) -> short convolution -> selective integrator -> join."""

    def __init__(self):
        super().__init__()
        from delrec.linear import Linear
        from delrec.neuron import BlockJoin, BlockNorm, SelectiveIntegrator, ShortConv
        self.first = BlockNorm(N)
        self.proj = torch.nn.ModuleList(Linear(N, 3 * N + 2 * S, binary_input=False) for _ in range(2))
        self.conv = torch.nn.ModuleList(ShortConv(N) for _ in range(2))
        self.core = torch.nn.ModuleList(SelectiveIntegrator(N, S) for _ in range(2))
        self.join = torch.nn.ModuleList(BlockJoin(N, "none", 0.5) for _ in range(2))
        self.head = torch.nn.Parameter(torch.randn(V, N) * 0.3)

    def forward(self, x, lengths=None):
        n = self.first(x, lengths)
        for proj, conv, core, join in zip(self.proj, self.conv, self.core, self.join):
            z, u, dt, bm, cm = proj(n).split([N, N, N, S, S], -1)
            if core.step_mode == "s":
                h = core(conv(z[0]), dt[0], bm[0], cm[0], u[0])[None]
            else:
                h = core(conv(z, lengths), dt, bm, cm, u, lengths)
            x, n = join(x, h, None, lengths)
        return n

    def loss(self, x, target, lengths=None, **kw):
        from delrec.vocab_loss import linear_cross_entropy
        return linear_cross_entropy(self(x, lengths), self.head, target, lengths=lengths, **kw)


def _reference(params, x, lengths, target):
    """The same network in float64 with autograd, on the CPU."""
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in params.items()}
    live = (torch.arange(T)[:, None] < lengths[None, :])[..., None]
    x = x.detach().double().cpu().requires_grad_(True)
    s = torch.where(live, x, torch.zeros_like(x))
    _, n = O.block_join(s, None, None, None, "none", None, p["first.weight"], 1e-5, True)
    for i in range(2):
        z, u, dt, bm, cm = (n @ p[f"proj.{i}.weight"].t() + p[f"proj.{i}.bias"]).split([N, N, N, S, S], -1)
        ext = torch.cat([torch.zeros(3, B, N, dtype=torch.float64), z])
        c = p[f"conv.{i}.bias"] + sum(p[f"conv.{i}.weight"][:, j] * ext[j:j + T] for j in range(4))
        c = c * torch.sigmoid(c)
        delta = torch.nn.functional.softplus(dt + p[f"core.{i}.dt_bias"])
        A = -torch.exp(p[f"core.{i}.A_log"])
        h, hs = torch.zeros(B, N, S, dtype=torch.float64), []
        for t in range(T):
            h = torch.exp(delta[t].unsqueeze(-1) * A) * h + (delta[t] * c[t]).unsqueeze(-1) * bm[t].unsqueeze(1)
            hs.append((h * cm[t].unsqueeze(1)).sum(-1) + p[f"core.{i}.D"] * c[t])
        y = torch.stack(hs) * u * torch.sigmoid(u)
        y = torch.where(live, y, torch.zeros_like(y))
        s, n = O.block_join(s, y, p[f"join.{i}.weight"], None, "none", p[f"join.{i}.scale"], p[f"join.{i}.next_weight"], 1e-5, True)
        s, n = torch.where(live, s, torch.zeros_like(s)), torch.where(live, n, torch.zeros_like(n))
    rows = (live[..., 0] & (target != -100)).flatten()
    loss = torch.nn.functional.cross_entropy((n @ p["head"].t()).flatten(0, 1)[rows], target.flatten()[rows])
    return loss, p, x


def _case(seed=3):
    torch.manual_seed(seed)
    model = Stack().cuda()
    x = torch.randn(T, B, N, device="cuda")
    target = torch.randint(0, V, (T, B), device="cuda")
    target[torch.rand(T, B, device="cuda") < 0.1] = -100
    return model, x, target, torch.tensor([T, 17, 1])


def test_training_pass():
    """The loss and every gradient against float64.  Relative to each tensor's largest entry: fp32 projections to 1e-5
    (their own tests' tolerance), three in a row on the longest path and as many again backward, so 1e-4."""
    model, x, target, lengths = _case()
    x.requires_grad_(True)
    loss = model.loss(x, target, lengths.cuda())
    params = dict(model.named_parameters())
    grads = torch.autograd.grad(loss, [x, *params.values()])
    ref, p, xr = _reference(params, x, lengths, target.cpu())
    want = torch.autograd.grad(ref, [xr, *p.values()])
    for got, w, name in zip((loss.detach(), *grads), (ref.detach(), *want), ("loss", "x", *params)):
        err = (got.double().cpu() - w).abs().max() / w.abs().max()
        assert err < 1e-4, f"{name}: {err:.2e}"


def test_streaming_is_the_whole_sequence():
    from delrec.utils import reset_states
    model, x, _, _ = _case()
    with torch.no_grad():
        whole = model(x)
        for m in (*model.core, *model.conv):
            m.step_mode = "s"
        for _ in range(2):
            reset_states(model)
            for t in range(T):
                torch.testing.assert_close(model(x[t:t + 1])[0], whole[t], rtol=1e-4, atol=1e-4)


def test_pieces_with_kept_state():
    from delrec.neuron import SelectiveIntegrator, ShortConv
    from delrec.utils import reset_states
    torch.manual_seed(1)
    x, dt, u = (torch.randn(T, B, N, device="cuda") for _ in range(3))
    bm, cm = (torch.randn(T, B, S, device="cuda") for _ in range(2))
    core, conv = SelectiveIntegrator(N, S, keep_state=True).cuda(), ShortConv(N, 5, keep_state=True).cuda()
    whole = core(conv(x), dt, bm, cm, u)
    for _ in range(2):
        reset_states(core)
        reset_states(conv)
        got = torch.cat([core(conv(x[a:b]), dt[a:b], bm[a:b], cm[a:b], u[a:b]) for a, b in ((0, 1), (1, 18), (18, T))])
        torch.testing.assert_close(got, whole, rtol=2 ** -18, atol=2 ** -18)


def test_module_layouts():
    from delrec.neuron import SelectiveIntegrator, ShortConv
    assert sorted(ShortConv(8).state_dict()) == ["bias", "weight"] and sorted(ShortConv(8, bias=False).state_dict()) == ["weight"]
    m = SelectiveIntegrator(8, 4)
    assert sorted(m.state_dict()) == ["A_log", "D", "dt_bias"] and m.v is None
    step = torch.nn.functional.softplus(m.dt_bias)
    assert (step > 0.99e-3).all() and (step < 0.101).all()
    for bad in (lambda: ShortConv(8, step_mode="x"), lambda: ShortConv(8, act="relu"), lambda: SelectiveIntegrator(8, step_mode="x")):
        with pytest.raises(ValueError):
            bad()


def test_zoo_losses_are_those_of_the_readout():
    """SNN.position_loss and distill_loss against the formed readout, loss and gradients, in float32: projections good
    to 1e-5 of the largest entry, and as much again for the logits' own sums."""
    from delrec import networks
    from model_configs import mem_config
    torch.manual_seed(0)
    model = networks.SNN(mem_config(hidden=[32], bias=True, T=16, B=4, C=8, K=50)).cuda()
    x = (torch.rand(16, 4, 8, device="cuda") < 0.4).float() * 2.5
    target = torch.randint(0, 50, (16, 4), device="cuda")
    idx = torch.rand(16, 4, 50, device="cuda").topk(5, -1).indices
    logits = torch.randn(16, 4, 5, device="cuda")
    p = torch.softmax(logits / 2, -1)

    def distilled(z):
        return 4 * (p * (p.log() - torch.log_softmax(z / 2, -1).gather(-1, idx))).sum(-1).mean()

    params = list(model.parameters())
    for got, want in ((model.position_loss(x, target), torch.nn.functional.cross_entropy(model(x).flatten(0, 1), target.flatten())),
                      (model.distill_loss(x, idx, logits, temperature=2.0), distilled(model(x)))):
        torch.testing.assert_close(got, want, rtol=2e-5, atol=2e-5)
        for a, b in zip(torch.autograd.grad(got, params), torch.autograd.grad(want, params)):
            assert (a - b).abs().max() <= 2e-5 * b.abs().max()


def _capture(fn):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_captured_training_pass():
    model, x, target, lengths = _case()
    lengths = lengths.cuda()
    params = list(model.parameters())

    def go():
        loss = model.loss(x, target, lengths)
        return (loss.detach(), *torch.autograd.grad(loss, params))

    graph, got = _capture(go)
    x.copy_(torch.randn_like(x))
    target.copy_(torch.randint(0, V, (T, B)))
    lengths.copy_(torch.tensor([5, T, 0]))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, go()):
        assert torch.equal(a, b)


def test_two_graphs_and_two_streams_at_once():
    """Two models' training passes, captured and replayed on two streams at once, and interleaved eagerly: each has
    the results it has alone."""
    cases = [_case(3), _case(4)]
    for model, *_ in cases:
        for proj in model.proj:
            proj.checkpoint8 = True       # the projections without it keep one workspace per stream, captured ones too

    def go(i):
        model, x, target, lengths = cases[i]
        loss = model.loss(x, target, lengths.cuda() if not torch.cuda.is_current_stream_capturing() else None, reduction="sum")
        return (loss.detach(), *torch.autograd.grad(loss, list(model.parameters())))

    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    want = [go(0), go(1)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(go(i))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(a, b)
    del got
    graphs = [_capture(lambda i=i: go(i)) for i in range(2)]
    for _ in range(4):
        for (graph, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for i, (_, out) in enumerate(graphs):
        model, x, target, _ = cases[i]
        loss = model.loss(x, target, reduction="sum")
        for a, b in zip(out, (loss.detach(), *torch.autograd.grad(loss, list(model.parameters())))):
            assert torch.equal(a, b)


def _calls():
    """name -> (callable, its tensors that may carry a gradient)"""
    from delrec.selective import selective_scan, selective_step
    from delrec.short_conv import short_conv, short_conv_step
    from delrec.vocab_loss import linear_cross_entropy, linear_distill
    r = lambda *s: torch.randn(*s, device="cuda")   # noqa: E731
    x, w, b, st = r(5, 2, 8), r(8, 4), r(8), r(3, 2, 8)
    dt, A, bm, cm, h0, D, gate, bias = r(5, 2, 8), -r(8, 4).exp(), r(5, 2, 4), r(5, 2, 4), r(2, 8, 4), r(8), r(5, 2, 8), r(8)
    head, hb = r(20, 8), r(20)
    t = torch.randint(0, 20, (5, 2), device="cuda")
    i, l = torch.randint(0, 20, (5, 2, 3), device="cuda"), r(5, 2, 3)
    return {
        "short_conv": (lambda x, w, b, st: short_conv(x, w, b, st), (x, w, b, st)),
        "short_conv_step": (lambda x, w, b, st: short_conv_step(x, w, b, st), (x[0], w, b, st)),
        "selective_scan": (lambda x, dt, A, bm, cm, h0, D, g, bias: selective_scan(x, dt, A, bm, cm, h0, D=D, gate=g, dt_bias=bias),
                           (x, dt, A, bm, cm, h0, D, gate, bias)),
        "selective_step": (lambda x, dt, A, bm, cm, h0, D, g, bias: selective_step(x, dt, A, bm, cm, h0, D=D, gate=g, dt_bias=bias),
                           (x[0], dt[0], A, bm[0], cm[0], h0, D, gate[0], bias)),
        "linear_cross_entropy": (lambda x, w, b: (linear_cross_entropy(x, w, t, b),), (x, head, hb)),
        "linear_distill": (lambda x, w, b: (linear_distill(x, w, i, l, b),), (x, head, hb)),
    }


@pytest.mark.parametrize("name", ["short_conv", "short_conv_step", "selective_scan", "selective_step", "linear_cross_entropy",
                                  "linear_distill"])
def test_forward_mode_derivatives_are_refused(name):
    import torch.autograd.forward_ad as fw
    fn, args = _calls()[name]
    want = fn(*args)
    with fw.dual_level():
        for k in range(len(args)):
            dual = [fw.make_dual(a, torch.ones_like(a)) if i == k else a for i, a in enumerate(args)]
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    fn(*dual)
        inside = fn(*args)
    for a, b, c in zip(fn(*args), want, inside):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("name", ["short_conv", "selective_scan", "linear_cross_entropy", "linear_distill"])
def test_second_derivatives_are_refused(name):
    fn, args = _calls()[name]
    args = [a.detach().requires_grad_(True) for a in args]
    out = fn(*args)[0]
    go = torch.randn_like(out).requires_grad_(True)
    (g,) = torch.autograd.grad(out, args[0], go, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_a_state_updated_in_place_is_seen_by_autograd():
    from delrec.selective import selective_step
    from delrec.short_conv import short_conv_step
    r = lambda *s: torch.randn(*s, device="cuda")   # noqa: E731
    for state, step in ((r(3, 2, 8), lambda s: short_conv_step(r(2, 8), r(8, 4), None, s, out=s)),
                        (r(2, 8, 4), lambda s: selective_step(r(2, 8), r(2, 8), -r(8, 4).exp(), r(2, 4), r(2, 4), s, out=s))):
        w = torch.randn_like(state).requires_grad_(True)
        saved = (state * w).sum()             # keeps state for w's gradient
        step(state)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            saved.backward()
        with torch.inference_mode():          # a streaming state has no version there
            step(torch.zeros_like(state))
    with pytest.raises(RuntimeError, match="teacher"):
        from delrec.vocab_loss import linear_distill
        linear_distill(r(2, 8), r(9, 8), torch.zeros(2, 1, dtype=torch.int32, device="cuda"), r(2, 1).requires_grad_(True))


@pytest.mark.parametrize("name", ["short_conv", "short_conv_step", "selective_scan", "selective_step", "linear_cross_entropy",
                                  "linear_distill"])
def test_calls_make_their_tensors_device_current(name, monkeypatch):
    fn, args = _calls()[name]
    train = name in ("short_conv", "selective_scan", "linear_cross_entropy", "linear_distill")
    args = [a.detach().requires_grad_(train) for a in args]

    def go():
        out = fn(*args)
        return [v.detach() for v in out] + (list(torch.autograd.grad(out[0], args[:2], torch.ones_like(out[0]))) if train else [])

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
    assert entered == ([0, 0] if train else [0])
    monkeypatch.undo()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_one_value_of_a_broadcast_input():
    """Inputs expanded along time and batch, and a gradient expanded from one value: the sum reaches the one."""
    from delrec.selective import selective_scan
    x = torch.randn(1, 1, 8, device="cuda", requires_grad=True)
    dt = torch.randn(9, 2, 8, device="cuda")
    A, bm = -torch.rand(8, 4, device="cuda") - 0.1, torch.randn(9, 2, 4, device="cuda")
    y, _ = selective_scan(x.expand(9, 2, 8), dt, A, bm, bm)
    (a,) = torch.autograd.grad(y.sum(), x)
    full = x.detach().expand(9, 2, 8).clone().requires_grad_(True)
    y2, _ = selective_scan(full, dt, A, bm, bm)
    (b,) = torch.autograd.grad(y2, full, torch.ones_like(y2))
    assert torch.equal(y, y2) and torch.equal(a, b.sum((0, 1), keepdim=True))


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements (4.3 GB each): the last rows are those of a call on them alone."""
    from delrec.selective import selective_scan
    from delrec.short_conv import short_conv
    Tb, Bb, Nb = 70000, 60, 520
    x = torch.empty(Tb, Bb, Nb, dtype=torch.bfloat16, device="cuda").normal_()
    assert x.numel() > 2 ** 31
    w = torch.randn(Nb, 4, device="cuda") * 0.5
    y, st = short_conv(x, w)
    one, last = short_conv(x[:, -1:].contiguous(), w)
    assert torch.equal(y[:, -1:], one) and torch.equal(st[:, -1:], last)
    del y
    bm = torch.empty(Tb, Bb, 4, dtype=torch.bfloat16, device="cuda").normal_()
    A = -torch.rand(Nb, 4, device="cuda") - 0.2
    y, hT = selective_scan(x, x, A, bm, bm)
    one, last = selective_scan(x[:, -1:].contiguous(), x[:, -1:], A, bm[:, -1:], bm[:, -1:])
    # the same sums cut in other places: fp32, then one bf16 step
    torch.testing.assert_close(y[:, -1:], one, rtol=2.0 ** -7, atol=2.0 ** -10)
    torch.testing.assert_close(hT[-1:], last, rtol=2.0 ** -15, atol=2.0 ** -15)


def test_backward_past_32_bits():
    from delrec.selective import selective_scan
    from delrec.short_conv import short_conv
    Tb, Bb, Nb = 4200, 1024, 512
    x = torch.empty(Tb, Bb, Nb, dtype=torch.bfloat16, device="cuda").normal_()
    w = torch.randn(Nb, 4, device="cuda") * 0.5
    g = torch.ones(1, 1, 1, dtype=torch.bfloat16, device="cuda").expand(Tb, Bb, Nb)
    xx = x.detach().requires_grad_(True)
    (dx,) = torch.autograd.grad(short_conv(xx, w)[0], xx, g)
    xs = x[:, -1:].clone().requires_grad_(True)
    (ds,) = torch.autograd.grad(short_conv(xs, w)[0], xs, g[:, -1:])
    assert torch.equal(dx[:, -1:], ds)
    del dx
    bm = torch.empty(Tb, Bb, 1, dtype=torch.bfloat16, device="cuda").normal_()
    A = -torch.rand(Nb, 1, device="cuda") - 0.2
    (dx,) = torch.autograd.grad(selective_scan(xx, x, A, bm, bm)[0], xx, g)
    (ds,) = torch.autograd.grad(selective_scan(xs, x[:, -1:], A, bm[:, -1:], bm[:, -1:])[0], xs, g[:, -1:])
    torch.testing.assert_close(dx[:, -1:], ds, rtol=2.0 ** -7, atol=2.0 ** -10)


def test_a_vocabulary_of_more_than_31_bits():
    """A weight of more than 2^31 elements: the loss, dx and the rows of dweight at its end."""
    from delrec.vocab_loss import linear_cross_entropy
    Vb, D, M = (1 << 21) + 77, 1040, 6
    w = torch.empty(Vb, D, dtype=torch.bfloat16, device="cuda").normal_(std=0.05).requires_grad_(True)
    assert w.numel() > 2 ** 31
    x = torch.randn(M, D, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    t = torch.tensor([0, Vb - 1, Vb - 2, 5, Vb // 2, Vb - 70], device="cuda")
    loss = linear_cross_entropy(x, w, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w))
    z = torch.cat([x.detach().float() @ w[a:a + (1 << 18)].detach().float().t() for a in range(0, Vb, 1 << 18)], 1)
    lse = torch.logsumexp(z, 1)
    want = (lse - z.gather(1, t[:, None])[:, 0]).sum()
    # (D / 16 + 12) 2 u of the logits' magnitudes (below 60) twice, 300 u a loss
    assert abs(loss.item() - want.item()) <= 6 * 2.0 ** -24 * (154 * 60 * 2 + 300)
    G = torch.softmax(z, 1)
    G[torch.arange(M), t] -= 1
    tail = slice(Vb - 100, Vb)
    ref = G[:, tail].double().t() @ x.detach().double()
    mag = G[:, tail].abs().double().t() @ x.detach().abs().double()
    # G rounded once to bf16, the sum once more
    assert ((dw[tail].double() - ref).abs() <= 2.0 ** -8 * 1.02 * (mag + ref.abs())).all()
    refx = sum(G[:, a:a + (1 << 18)].double() @ w[a:a + (1 << 18)].detach().double() for a in range(0, Vb, 1 << 18))
    magx = sum(G[:, a:a + (1 << 18)].abs().double() @ w[a:a + (1 << 18)].detach().abs().double() for a in range(0, Vb, 1 << 18))
    assert ((dx.double() - refx).abs() <= 2.0 ** -8 * 1.02 * (magx + refx.abs())).all()
