"""The block norms (delrec.block_norm) against float64 autograd over their formula.

Tolerance: a row's sum of N products is good to 64 u of its terms' magnitudes (at most 32 in a
thread, a shuffle tree, 16 warps), a gate to 8 u, and every output is a sum of terms that go
through at most two such sums and a dozen products: C = 256 units u = 2^-24 of the summed
magnitudes of the terms, plus half a step of the stored type."""

import pytest
import torch

from oracle import sequence_oracle as O
from sequence_cases import within

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
C = 256 * O.U
EPS = 1e-5


def _inputs(T, B, N, dtype, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + T * 31 + B * 17 + N)
    r = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    return dict(x=(1.5 * r(T, B, N)).to(dtype), y=(0.7 * r(T, B, N)).to(dtype), u=(2 * r(T, B, N)).to(dtype),
                w=1 + 0.1 * r(N), scale=0.5 + 0.1 * r(N), nw=1 + 0.1 * r(N), gx=r(T, B, N).to(dtype),
                gn=r(T, B, N).to(dtype))


def _reference(c, kind, has_y, has_next, eps, live):
    """Outputs and gradients in float64 (rows that are not live left out), and their bounds."""
    d = {k: (v.double() if v is not None else None) for k, v in c.items()}
    T, B, N = d["x"].shape
    rows = lambda v: None if v is None else v[live]      # noqa: E731
    for k in ("x", "y", "u", "gx", "gn"):
        d[k] = rows(d[k])
    leaves = [k for k in ("x", "y", "u", "w", "scale", "nw") if d[k] is not None]
    for k in leaves:
        d[k].requires_grad_(True)
    new, n = O.block_join(d["x"], d["y"] if has_y else None, d["w"], d["u"], kind, d["scale"], d["nw"], eps, has_next)
    outs = [t for t in (new, n) if t is not None]
    gs = ([d["gx"]] if has_y else []) + ([d["gn"]] if has_next else [])
    grads = dict(zip(leaves, torch.autograd.grad(outs, [d[k] for k in leaves], gs, allow_unused=True)))
    # magnitudes of the terms
    with torch.no_grad():
        A = lambda v: 0.0 if v is None else v.abs()      # noqa: E731
        one = torch.ones(N, dtype=torch.float64)
        w, sc, nw = (A(d[k]) if d[k] is not None else one for k in ("w", "scale", "nw"))
        err = {}
        if has_y:
            ry = 1 / (d["y"].pow(2).mean(-1, keepdim=True) + eps).sqrt()
            yh = d["y"].abs() * ry
            if d["u"] is not None and kind != "none":
                s = O.sigmoid(d["u"])
                so = O.sigmoid(-d["u"])
                a, da = (s, s * so) if kind == "sigmoid" else ((s * d["u"]).abs(),
                                                                   s * (1 + d["u"].abs() * so))
            else:
                a, da = torch.ones_like(yh), None
            mag = d["x"].abs() + sc * a * yh * w
            err["new"] = C * mag
            val = new
        else:
            mag, val = d["x"].abs(), d["x"]
        G = d["gx"].abs() if has_y else torch.zeros_like(mag)
        if has_next:
            rx = 1 / (val.pow(2).mean(-1, keepdim=True) + eps).sqrt()
            xm = mag * rx                                 # the magnitude that xh comes from
            spread = (xm.pow(2).mean(-1, keepdim=True)).sqrt()   # what an error of x' does to rx, relative
            xm = xm + xm * spread
            err["n"] = C * xm * nw
            v = d["gn"].abs() * nw
            m = (v * xm).mean(-1, keepdim=True)
            G = G + rx * (v + xm * m) * (1 + spread)
            err["nw"] = C * (d["gn"].abs() * xm).sum(0) * (1 + len(xm) / 256)
        err["x"] = C * G
        if has_y:
            err["w"] = C * sc * (G * a * yh).sum(0) * (1 + len(G) / 256)
            err["scale"] = C * w * (G * a * yh).sum(0) * (1 + len(G) / 256)
            v = G * sc * a * w
            err["y"] = C * ry * (v + yh * (v * yh).mean(-1, keepdim=True))
            if da is not None:
                err["u"] = C * G * sc * yh * w * da

    def full(v):
        if v is None or v.dim() == 1:
            return v
        out = torch.zeros(T, B, N, dtype=torch.float64)
        out[live] = v.detach()
        return out

    res = {"new": full(new), "n": full(n), **{k: full(v) for k, v in grads.items()}}
    return res, {k: full(v) for k, v in err.items()}


def _check(c, kind="sigmoid", has_next=True, lengths=None, eps=EPS, weights=True):
    from delrec.block_norm import block_join
    c = dict(c)
    if not weights:
        c["w"] = c["scale"] = c["nw"] = None
    if kind is None:
        c["u"] = None
    if not has_next:
        c["nw"] = c["gn"] = None
    T, B, N = c["x"].shape
    live = torch.ones(T, B, dtype=torch.bool)
    if lengths is not None:
        live = torch.arange(T)[:, None] < lengths[None, :]
    d = {k: None if v is None else v.cuda() for k, v in c.items()}
    leaves = [k for k in ("x", "y", "u", "w", "scale", "nw") if d[k] is not None]
    for k in leaves:
        d[k].requires_grad_(True)
    new, n = block_join(d["x"], d["y"], d["w"], gate=d["u"], gate_act=kind or "sigmoid", scale=d["scale"],
                        next_weight=d["nw"], next_norm=has_next, eps=eps,
                        lengths=None if lengths is None else lengths.cuda())
    outs = [t for t in (new, n) if t is not None]
    grads = dict(zip(leaves, torch.autograd.grad(outs, [d[k] for k in leaves],
                                                 [t for t in (d["gx"], d["gn"]) if t is not None])))
    ref, err = _reference(c, kind or "none", True, has_next, eps, live)
    within(new, ref["new"], err["new"], "x'")
    if has_next:
        within(n, ref["n"], err["n"], "n")
    else:
        assert n is None
    for k in leaves:
        within(grads[k], ref[k], err[k], "d" + k)
    return [t.detach() for t in outs], grads


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,B,N", [(1, 1, 1), (1, 2, 4), (2, 3, 31), (3, 2, 64), (1, 5, 100), (4, 3, 128), (2, 2, 130),
                                   (3, 3, 512), (2, 2, 700), (2, 1, 1022), (1, 2, 2048), (2, 1, 2049)])
def test_join(T, B, N, dtype):
    _check(_inputs(T, B, N, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N", [4096, 5000, 8190, 8191, 8192, 12000, 16383, 16384])
def test_join_wide(N, dtype):
    _check(_inputs(2, 2, N, dtype))


@pytest.mark.parametrize("weights", [True, False])
@pytest.mark.parametrize("has_next", [True, False])
@pytest.mark.parametrize("kind", [None, "none", "sigmoid", "silu"])
def test_join_forms(kind, has_next, weights):
    c = _inputs(5, 3, 96, F32)
    if kind == "none":
        c["u"] = None      # a gate with the activation "none" is not read
    _check(c, kind, has_next, weights=weights)


@pytest.mark.parametrize("kind", ["sigmoid", "silu"])
def test_ragged_padding_is_not_read(kind):
    for N in (33, 256):
        c = _inputs(9, 5, N, F32)
        lengths = torch.tensor([0, 9, 1, 4, 8])
        outs, grads = _check(c, kind, lengths=lengths)
        for k in ("x", "y", "u", "gx", "gn"):
            for b in range(5):
                c[k][int(lengths[b]):, b] = float("nan")
        from delrec.block_norm import block_join
        d = {k: v.cuda() for k, v in c.items()}
        leaves = ("x", "y", "u", "w", "scale", "nw")
        for k in leaves:
            d[k].requires_grad_(True)
        got = block_join(d["x"], d["y"], d["w"], gate=d["u"], gate_act=kind, scale=d["scale"], next_weight=d["nw"],
                         eps=EPS, lengths=lengths.int().cuda())
        g2 = torch.autograd.grad(got, [d[k] for k in leaves], (d["gx"], d["gn"]))
        for a, b in zip(got, outs):
            assert torch.equal(a, b)
        for a, k in zip(g2, leaves):
            assert torch.equal(a, grads[k])


def test_all_rows_empty():
    from delrec.block_norm import block_join
    c = {k: v.cuda().requires_grad_(True) for k, v in _inputs(4, 2, 40, F32).items()}
    new, n = block_join(c["x"], c["y"], c["w"], gate=c["u"], scale=c["scale"], next_weight=c["nw"],
                        lengths=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert not new.any() and not n.any()
    for g in torch.autograd.grad((new, n), [c[k] for k in ("x", "y", "u", "w", "scale", "nw")], (c["gx"], c["gn"])):
        assert not g.any()


@pytest.mark.parametrize("N", [1, 33, 512, 3000])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_norm_alone(N, dtype):
    from delrec.block_norm import block_norm
    c = _inputs(3, 2, N, dtype)
    for weight in (True, False):
        x = c["x"].cuda().requires_grad_(True)
        w = c["nw"].cuda().requires_grad_(True) if weight else None
        n = block_norm(x, w, eps=EPS)
        leaves = [t for t in (x, w) if t is not None]
        grads = torch.autograd.grad(n, leaves, c["gn"].cuda())
        k = dict(x=c["x"], y=None, u=None, w=None, scale=None, nw=c["nw"] if weight else None, gx=None, gn=c["gn"])
        ref, err = _reference(k, "none", False, True, EPS, torch.ones(3, 2, dtype=torch.bool))
        within(n, ref["n"], err["n"], "n")
        within(grads[0], ref["x"], err["x"], "dx")
        if weight:
            within(grads[1], ref["nw"], err["nw"], "dw")


def test_zero_rows_and_saturated_gates():
    c = _inputs(4, 2, 64, F32)
    c["y"][0, 0] = 0
    c["x"][1, 1] = 0
    c["y"][1, 1] = 0
    c["u"][2] = 100.0
    c["u"][3] = -100.0
    for kind in ("sigmoid", "silu"):
        _check(c, kind)


def test_large_values():
    """Rows whose mean square is far from 1: 1e15 squared fits fp32, fp16's largest does too."""
    c = _inputs(3, 2, 64, F32)
    c["x"] *= 1e15
    c["y"] *= 1e15
    _check(c)
    c = _inputs(3, 2, 64, F16)
    c["y"] = (c["y"].float() * 2e4).clamp(-6e4, 6e4).half()
    c["x"] = (c["x"].float() * 1e4).clamp(-6e4, 6e4).half()
    _check(c)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(dtype):
    """Batch-major storage, slices at odd offsets, expanded rows: the bits of contiguous tensors."""
    from delrec.block_norm import block_join
    T, B, N = 6, 3, 64
    g = torch.Generator().manual_seed(3)
    big = torch.randn(B, T, 5 * N + 9, generator=g).to(dtype).cuda()
    v = [big[:, :, i * N + i:(i + 1) * N + i].transpose(0, 1) for i in range(5)]
    w = torch.randn(N, generator=g).cuda()

    def go(x, y, u, gx, gn):
        x, y, u = (t.detach().requires_grad_(True) for t in (x, y, u))
        ww = w.clone().requires_grad_(True)
        o = block_join(x, y, ww, gate=u, scale=w, next_weight=w)
        return (*o, *torch.autograd.grad(o, (x, y, u, ww), (gx, gn)))

    base = go(*(t.contiguous() for t in v))
    strided = v[1].transpose(1, 2).contiguous().transpose(1, 2)
    for got in (go(*v), go(v[0], strided, *v[2:])):
        for a, b in zip(got, base):
            torch.testing.assert_close(a, b, rtol=2.0 ** -7 if dtype == BF16 else 2.0 ** -18, atol=2.0 ** -18)
    row = v[1][2:3, 1:2].expand(T, B, N)
    for a, b in zip(go(v[0], row, *v[2:]), go(v[0], row.contiguous(), *v[2:])):
        torch.testing.assert_close(a, b, rtol=2.0 ** -7 if dtype == BF16 else 2.0 ** -18, atol=2.0 ** -18)


def test_many_rows_sum_the_weight_gradients():
    T, B, N = 60, 80, 64
    c = _inputs(T, B, N, F32)
    _check(c)


def test_gradients_by_differences():
    from delrec.block_norm import block_join
    c = _inputs(4, 3, 48, F32)
    keys = ("x", "y", "u", "w", "scale", "nw")
    d = {k: v.cuda() for k, v in c.items()}
    for k in keys:
        d[k].requires_grad_(True)
    o = block_join(d["x"], d["y"], d["w"], gate=d["u"], gate_act="silu", scale=d["scale"], next_weight=d["nw"], eps=EPS)
    grads = torch.autograd.grad(o, [d[k] for k in keys], (d["gx"], d["gn"]))

    def loss(v):
        new, n = O.block_join(v["x"], v["y"], v["w"], v["u"], "silu", v["scale"], v["nw"], EPS, True)
        return (new * c["gx"].double()).sum() + (n * c["gn"].double()).sum()

    base = {k: c[k].double() for k in keys}
    g = torch.Generator().manual_seed(2)
    for k, grad in zip(keys, grads):
        v = torch.randn(base[k].shape, generator=g, dtype=torch.float64)
        num = (loss({**base, k: base[k] + 1e-5 * v}) - loss({**base, k: base[k] - 1e-5 * v})) / 2e-5
        t = grad.double().cpu() * v
        assert abs(num - t.sum()) < 1e-5 * t.abs().sum()


def test_partial_gradients_and_repeat():
    from delrec.block_norm import block_join
    c = {k: v.cuda() for k, v in _inputs(6, 4, 96, F32).items()}
    keys = ("x", "y", "u", "w", "scale", "nw")

    def go(want, outs="both"):
        t = {k: c[k].detach().requires_grad_(k in want) for k in keys}
        new, n = block_join(t["x"], t["y"], t["w"], gate=t["u"], scale=t["scale"], next_weight=t["nw"])
        o, g = {"both": ((new, n), (c["gx"], c["gn"])), "new": ((new,), (c["gx"],)), "n": ((n,), (c["gn"],))}[outs]
        r = torch.autograd.grad(o, [t[k] for k in want], g, allow_unused=True)
        return dict(zip(want, r))

    full = go(keys)
    for k in keys:
        assert torch.equal(go((k,))[k], full[k])
    a, b = go(keys, "new"), go(keys, "n")
    for k in keys:
        s = (a[k] if a[k] is not None else 0) + b[k]
        torch.testing.assert_close(s, full[k], rtol=2 ** -16, atol=2 ** -16)
    assert a["nw"] is None or not a["nw"].any()


@pytest.mark.parametrize("shape", [(0, 2, 5), (4, 0, 5), (4, 2, 0)])
def test_empty(shape):
    from delrec.block_norm import block_join
    t = [torch.randn(shape, device="cuda", requires_grad=True) for _ in range(3)]
    w = torch.ones(shape[-1], device="cuda", requires_grad=True)
    new, n = block_join(t[0], t[1], w, gate=t[2], next_weight=w)
    g = torch.autograd.grad((new, n), (*t, w), (torch.ones_like(new), torch.ones_like(n)))
    assert new.shape == n.shape == shape and not g[3].any()


def test_captured_in_a_graph():
    from delrec.block_norm import block_join
    c = {k: v.cuda() for k, v in _inputs(30, 4, 96, F32).items()}

    def go():
        t = {k: c[k].detach().requires_grad_(True) for k in ("x", "y", "u", "w")}
        o = block_join(t["x"], t["y"], t["w"], gate=t["u"], scale=c["scale"], next_weight=c["nw"])
        return (*(v.detach() for v in o), *torch.autograd.grad(o, list(t.values()), (c["gx"], c["gn"])))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        go()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(go())
        graphs.append(g)
    for k, v in _inputs(30, 4, 96, F32, seed=5).items():
        c[k].copy_(v.cuda())
    for g in graphs:
        g.replay()
    want = go()
    torch.cuda.synchronize()
    for got in outs:
        for a, b in zip(got, want):
            assert torch.equal(a, b)
