"""The selective scan and its step against their formulas in float64."""

import pytest
import torch

from sequence_cases import within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = dict(x="dx", dt="ddt", A="dA", Bm="dB", Cm="dC", h0="dh0", D="dD", gate="dgate", dt_bias="dbias")

# T, B, N, S, G, options ("0": h0, "D", "g": gate, "b": dt_bias, "n": no softplus, "r": resets), lengths
CASES = [(1, 1, 1, 1, 1, "", None), (1, 2, 8, 16, 1, "0Dgb", None), (9, 2, 5, 3, 1, "0Dgbr", [9, 0]),
         (17, 3, 36, 16, 1, "0Dgbr", [17, 1, 8]), (24, 2, 70, 24, 2, "0gb", [24, 23]), (33, 1, 12, 5, 3, "Dgn", None),
         (20, 2, 20, 64, 1, "0Dgbr", [11, 20]), (16, 1, 9, 128, 1, "0Dg", None), (12, 2, 10, 100, 2, "gbr", [12, 5]),
         (40, 1, 132, 8, 1, "0D", None), (31, 2, 66, 2, 1, "0Dgb", None), (300, 1, 20, 16, 1, "0Dgbr", [270]),
         (259, 2, 16, 4, 2, "0Dgb", [259, 130]), (400, 1, 6, 40, 1, "0gr", None)]


def _make(case, dtype, seed=0):
    T, B, N, S, G, opt, lengths = case
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    d = dict(x=rnd(T, B, N).to(dtype), dt=(rnd(T, B, N) * 0.5 - (0.0 if "b" in opt else 2.0)).to(dtype),
             A=-(torch.rand(N, S, generator=g) * S + 0.2), Bm=rnd(T, B, G, S).to(dtype), Cm=rnd(T, B, G, S).to(dtype),
             h0=rnd(B, N, S) if "0" in opt else None, D=rnd(N) if "D" in opt else None,
             gate=rnd(T, B, N).to(dtype) if "g" in opt else None, dt_bias=rnd(N) - 2.0 if "b" in opt else None,
             softplus="n" not in opt, lengths=torch.tensor(lengths, dtype=torch.int32) if lengths else None,
             resets=torch.rand(T, B, generator=g) < 0.15 if "r" in opt else None)
    if "n" in opt:
        d["dt"] = (rnd(T, B, N).abs() * 0.3).to(dtype)
    return d, rnd(T, B, N).to(dtype), rnd(B, N, S)


def _call(c):
    from delrec.selective import selective_scan
    return selective_scan(c["x"], c["dt"], c["A"], c["Bm"], c["Cm"], c["h0"], D=c["D"], gate=c["gate"],
                          dt_bias=c["dt_bias"], softplus=c["softplus"], lengths=c["lengths"], resets=c["resets"])


def _cuda(d):
    return {k: v.cuda() if torch.is_tensor(v) else v for k, v in d.items()}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_against_float64(case, dtype):
    from oracle import selective_oracle as O
    d, gy, gh = _make(case, dtype)
    ref = O.selective(**d, gy=gy, ghT=gh)
    c = _cuda(d)
    if c["lengths"] is not None:           # what stands past a length is not read
        past = torch.arange(case[0], device="cuda")[:, None] >= c["lengths"][None]
        for k in ("x", "dt", "gate", "Bm", "Cm"):
            if c[k] is not None:
                m = past.view(*past.shape, *[1] * (c[k].dim() - 2))
                c[k] = torch.where(m, torch.full_like(c[k], float("nan")), c[k])
        gy = torch.where(past.cpu().unsqueeze(-1), torch.full_like(gy, float("inf")), gy)
    leaves = [k for k in NAMES if c[k] is not None]
    for k in leaves:
        c[k].requires_grad_(True)
    y, hT = _call(c)
    within(y, ref["y"], ref["e_y"], "y")
    within(hT, ref["hT"], ref["e_hT"], "hT")
    grads = torch.autograd.grad((y, hT), [c[k] for k in leaves], (gy.cuda(), gh.cuda()))
    for k, v in zip(leaves, grads):
        within(v, ref[NAMES[k]], ref["e_" + NAMES[k]], NAMES[k])
    with torch.no_grad():
        for a, b in zip(_call(c), (y, hT)):
            assert torch.equal(a, b)


def test_gradient_against_differences():
    """The float64 oracle's gradients are those of its own forward pass."""
    from oracle import selective_oracle as O
    d, gy, gh = _make((7, 2, 4, 3, 2, "0Dgbr", [7, 5]), torch.float32, 3)
    d = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in d.items()}
    gy, gh = gy.double(), gh.double()
    ref = O.selective(**d, gy=gy, ghT=gh)
    value = lambda e: (lambda r: (r["y"] * gy).sum() + (r["hT"] * gh).sum())(O.selective(**e))   # noqa: E731
    for k, name in NAMES.items():
        v = torch.randn(d[k].shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
        diff = (value({**d, k: d[k] + 1e-5 * v}) - value({**d, k: d[k] - 1e-5 * v})) / 2e-5
        assert abs(diff - (ref[name] * v).sum()) <= 1e-7 * (1 + (ref[name] * v).abs().sum()), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,S,G", [(8, 16, 1), (10, 3, 2), (3, 128, 1), (36, 33, 4), (5, 1, 1)])
def test_step(N, S, G, dtype):
    """Single steps against float64, in place, with rows that are not active."""
    from delrec.selective import selective_step
    from oracle import selective_oracle as O
    d, _, _ = _make((4, 3, N, S, G, "0Dgb", None), dtype, 1)
    ref = O.selective(**d)
    c = _cuda(d)
    kw = dict(D=c["D"], dt_bias=c["dt_bias"])
    state = c["h0"].clone()
    for t in range(4):
        y, out = selective_step(c["x"][t], c["dt"][t], c["A"], c["Bm"][t], c["Cm"][t], state, gate=c["gate"][t], out=state, **kw)
        assert out is state
        within(y, ref["y"][t], ref["e_y"][t], f"y {t}")
    within(state, ref["hT"], ref["e_hT"], "state")
    args = c["x"][0], c["dt"][0], c["A"], c["Bm"][0], c["Cm"][0]
    active = torch.tensor([False, True, False], device="cuda")
    y, nxt = selective_step(*args, state, gate=c["gate"][0], active=active, **kw)
    full, moved = selective_step(*args, state, gate=c["gate"][0], **kw)
    assert torch.equal(nxt[[0, 2]], state[[0, 2]]) and not y[[0, 2]].any()
    assert torch.equal(nxt[1], moved[1]) and torch.equal(y[1], full[1])
    # no state: zeros; a state at an odd address
    none = selective_step(*args, **kw)
    zero = selective_step(*args, torch.zeros_like(state), **kw)
    odd = torch.zeros(state.numel() + 1, device="cuda")[1:].view(state.shape)
    for v in (zero, selective_step(*args, odd, **kw), selective_step(*args, odd, out=odd, **kw)):
        assert torch.equal(none[0], v[0]) and torch.equal(none[1], v[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Batch-major tensors, strided channels, odd addresses and (T, B, S) inputs give the same numbers."""
    d, gy, gh = _make((21, 3, 24, 8, 1, "0Dgb", None), dtype)
    base = _cuda(d)
    gy, gh = gy.cuda(), gh.cuda()
    keys = ("x", "dt", "gate", "Bm", "Cm")

    def go(**kw):
        c = {**base, **kw}
        c.update({k: c[k].detach().requires_grad_(True) for k in keys})
        y, hT = _call(c)
        return [y, hT, *torch.autograd.grad((y, hT), [c[k] for k in keys], (kw.get("gy", gy), gh))]

    want = go()
    forms = [lambda v: v.transpose(0, 1).contiguous().transpose(0, 1), lambda v: torch.stack([v, v], -1)[..., 0],
             lambda v: torch.cat([v.new_zeros(1), v.flatten()])[1:].view(v.shape)]
    for form in forms:
        for k in keys:
            for a, b in zip(go(**{k: form(base[k])}), want):
                assert torch.equal(a, b), k
    got = go(Bm=base["Bm"][:, :, 0], Cm=base["Cm"][:, :, 0])
    assert got[5].shape == (21, 3, 8)
    for a, b in zip(got, want):
        assert torch.equal(a, b.view(a.shape))


def test_pieces_give_the_whole():
    d, _, _ = _make((40, 2, 20, 16, 1, "0Dgb", None), torch.float32)
    c = _cuda(d)
    y, hT = _call(c)
    cut = lambda a, b, **kw: {**c, **{k: c[k][a:b] for k in ("x", "dt", "gate", "Bm", "Cm")}, **kw}   # noqa: E731
    y1, h1 = _call(cut(0, 13))
    y2, h2 = _call(cut(13, 40, h0=h1))
    assert torch.equal(torch.cat([y1, y2]), y) and torch.equal(h2, hT)


def test_infinite_states_do_not_pass_a_reset():
    T, N, S = 40, 8, 4
    d, gy, gh = _make((T, 1, N, S, 1, "Dgb", None), torch.float32)
    c = _cuda(d)
    c["h0"] = torch.full((1, N, S), float("inf"), device="cuda")
    c["resets"] = torch.zeros(T, 1, dtype=torch.bool, device="cuda")
    c["resets"][5] = True
    for k in ("x", "dt"):
        c[k].requires_grad_(True)
    y, hT = _call(c)
    assert torch.isfinite(y[5:]).all() and torch.isfinite(hT).all() and not torch.isfinite(y[:5]).any()
    gy = gy.cuda()
    gy[:5] = 0
    dx, = torch.autograd.grad((y, hT), (c["x"],), (gy, gh.cuda()))
    assert torch.isfinite(dx[5:]).all()


def test_empty_sequences():
    from delrec.selective import selective_scan
    A, Dv = torch.full((6, 4), -1.0, device="cuda", requires_grad=True), torch.ones(6, device="cuda", requires_grad=True)
    for T, B in ((0, 2), (3, 0)):
        x = torch.randn(T, B, 6, device="cuda", requires_grad=True)
        bm = torch.randn(T, B, 4, device="cuda", requires_grad=True)
        h0 = torch.randn(B, 6, 4, device="cuda", requires_grad=True)
        y, hT = selective_scan(x, x, A, bm, bm, h0, D=Dv)
        assert y.shape == x.shape and torch.equal(hT, h0)
        grads = torch.autograd.grad((y, hT), (x, A, bm, Dv, h0), (torch.ones_like(y), torch.full_like(hT, 3.0)))
        assert not grads[1].any() and not grads[3].any() and torch.equal(grads[4], torch.full_like(h0, 3.0))


def test_one_of_two_gradients_and_of_one_input():
    from oracle import selective_oracle as O
    d, gy, gh = _make((19, 2, 12, 16, 1, "0Dgb", None), torch.float32)
    for use in ("y", "hT"):
        ref = O.selective(**d, **(dict(gy=gy) if use == "y" else dict(ghT=gh)))
        for k in ("x", "A", "Bm", "h0", "dt_bias"):
            c = _cuda(d)
            c[k].requires_grad_(True)
            y, hT = _call(c)
            (v,) = torch.autograd.grad(y if use == "y" else hT, c[k], (gy if use == "y" else gh).cuda())
            within(v, ref[NAMES[k]], ref["e_" + NAMES[k]], f"{NAMES[k]} of {use}")


@pytest.mark.parametrize("N,S,G,B", [(5, 4, 1, 31001), (512, 8, 1, 303), (700, 24, 2, 57), (40, 64, 4, 501), (33, 128, 3, 301),
                                     (16, 12, 1, 5003), (6000, 16, 1, 31)])
def test_step_of_many_sequences(N, S, G, B):
    """More states than threads: the states of the same calls on few sequences, bit for bit, and their
    outputs but for the order of a sum of S products."""
    from delrec.selective import selective_step
    g = torch.Generator().manual_seed(N)
    rnd = lambda *s: torch.randn(*s, generator=g).cuda()   # noqa: E731
    x, dt, gate = rnd(B, N), rnd(B, N), rnd(B, N)
    A, Bm, C, D, bias = -rnd(N, S).abs(), rnd(B, G, S), rnd(B, G, S), rnd(N), rnd(N)
    state = rnd(B, N, S)
    active = (torch.rand(B, generator=g) < 0.8).cuda()
    x[~active] = float("nan")               # what does not count is not read
    kw = dict(D=D, dt_bias=bias)
    few = max(1, B // 40)
    parts = [selective_step(x[i:i + few], dt[i:i + few], A, Bm[i:i + few], C[i:i + few], state[i:i + few], gate=gate[i:i + few],
                            active=active[i:i + few], **kw) for i in range(0, B, few)]
    y, nxt = (torch.cat(v) for v in zip(*parts))
    mag = (C.abs().repeat_interleave(N // G, 1) * nxt.abs()).sum(-1) + (D * x).abs()
    tol = torch.where(active[:, None], (S + 2) * 2.0 ** -23 * mag * gate.abs(), torch.zeros_like(y))
    for out in (None, state.clone()):
        got, h = selective_step(x, dt, A, Bm, C, state if out is None else out, gate=gate, active=active, out=out, **kw)
        assert torch.equal(h, nxt)
        assert ((got - y).abs() <= tol).all()
        assert torch.equal(h[~active], state[~active]) and (got[~active] == 0).all()
