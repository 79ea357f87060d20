"""The selective scan at decays without bounds and with many channels to a sequence."""

import pytest
import torch

from sequence_cases import within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
KEYS = ("x", "dt", "A", "Bm", "Cm", "h0", "D", "gate", "dt_bias")


def _inputs(T, B, N, S, dtype, lengths, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    d = dict(x=rnd(T, B, N).to(dtype), dt=rnd(T, B, N).to(dtype), A=-rnd(N, S).abs() - 0.1, Bm=rnd(T, B, S).to(dtype),
             Cm=rnd(T, B, S).to(dtype), h0=rnd(B, N, S), D=rnd(N), gate=rnd(T, B, N).to(dtype), dt_bias=rnd(N))
    d = {k: v.cuda() for k, v in d.items()}
    return d, torch.tensor(lengths, device="cuda") if lengths else None, rnd(T, B, N).to(dtype).cuda(), rnd(B, N, S).cuda()


def _run(d, lengths, gy, gh, **kw):
    from delrec.selective import selective_scan
    c = {k: v.detach().clone().requires_grad_(True) for k, v in d.items()}
    y, hT = selective_scan(c["x"], c["dt"], c["A"], c["Bm"], c["Cm"], c["h0"], D=c["D"], gate=c["gate"], dt_bias=c["dt_bias"],
                           lengths=lengths, **kw)
    return [y, hT, *torch.autograd.grad((y, hT), [c[k] for k in KEYS], (gy, gh))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,N,S,lengths", [(13, 2, 6, 5, [13, 3]), (8, 1, 4, 16, None), (9, 3, 40, 4, [0, 9, 1]),
                                             (300, 2, 8, 16, [300, 77]), (515, 1, 5, 1, None)])
def test_a_decay_of_minus_infinity_drops_the_state(T, B, N, S, lengths, dtype):
    """A = -inf (what -exp(A_log) gives past A_log = 88.7) is a decay of 0 in every step there is: the bits of A = -1e30,
    whose decay is 0 as well, and no trace in the steps that there are not."""
    d, lengths, gy, gh = _inputs(T, B, N, S, dtype, lengths)
    hit = torch.rand(N, S, generator=torch.Generator().manual_seed(1)).cuda() < 0.4
    hit[0, 0] = True
    big = dict(d, A=torch.where(hit, torch.full_like(d["A"], -1e30), d["A"]))
    inf = dict(d, A=torch.where(hit, torch.full_like(d["A"], -float("inf")), d["A"]))
    for got, want, name in zip(_run(inf, lengths, gy, gh), _run(big, lengths, gy, gh), ("y", "hT") + KEYS):
        assert torch.isfinite(want).all() and torch.equal(got, want), name
    # by the formula: such a state is the last step's input alone, or the first state where there is no step
    hT = _run(inf, lengths, gy, gh)[1].detach().double()
    for b in range(B):
        n = T if lengths is None else int(lengths[b])
        if n == 0:
            assert torch.equal(hT[b], d["h0"][b].double())
            continue
        delta = torch.nn.functional.softplus(d["dt"][n - 1, b].double() + d["dt_bias"].double())
        want = (delta * d["x"][n - 1, b].double())[:, None] * d["Bm"][n - 1, b].double()
        # delta good to (10 + |z|) u, three products
        assert ((hT[b] - want).abs()[hit] <= (32 * 2.0 ** -24 * want.abs())[hit] + 2.0 ** -140).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,N,S,G,launches", [(2, 900, 60, 128, 1, 2), (2, 1800, 40, 128, 2, 2), (9, 1800, 20, 70, 1, 2),
                                                (1, 4000, 33, 100, 1, 2), (1, 4000, 33, 40, 1, 1)])
def test_sums_over_many_tiles_of_channels(T, B, N, S, G, launches, dtype):
    """More tiles of channels than dB and dC have places for their sums: two launches add them up."""
    from delrec import _lib
    from delrec.selective import selective_scan
    from oracle import selective_oracle as O
    g = torch.Generator().manual_seed(6)
    rnd = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    d = dict(x=rnd(T, B, N).to(dtype), dt=(rnd(T, B, N) - 2).to(dtype), A=-rnd(N, S).abs() - 0.1, Bm=rnd(T, B, G, S).to(dtype),
             Cm=rnd(T, B, G, S).to(dtype), D=rnd(N), lengths=torch.randint(0, T + 1, (B,), generator=g))
    gy, gh = rnd(T, B, N).to(dtype), rnd(B, N, S)
    ref = O.selective(**d, gy=gy, ghT=gh)
    c = {k: v.cuda() for k, v in d.items()}
    leaves = ["x", "dt", "A", "Bm", "Cm", "D"]
    for k in leaves:
        c[k].requires_grad_(True)
    y, hT = selective_scan(c["x"], c["dt"], c["A"], c["Bm"], c["Cm"], D=c["D"], lengths=c["lengths"])
    before = _lib.launch_count()
    grads = torch.autograd.grad((y, hT), [c[k] for k in leaves], (gy.cuda(), gh.cuda()), retain_graph=True)
    assert _lib.launch_count() - before == launches + 3        # sums of dA, dD; dB and dC
    for k, v in zip(leaves, grads):
        name = dict(x="dx", dt="ddt", A="dA", Bm="dB", Cm="dC", D="dD")[k]
        within(v, ref[name], ref["e_" + name], name)
    # one of the two, and neither: the same numbers, and one launch for neither
    (dB,) = torch.autograd.grad((y, hT), c["Bm"], (gy.cuda(), gh.cuda()), retain_graph=True)
    assert torch.equal(dB, grads[3])
    y, hT = selective_scan(c["x"], c["dt"].detach(), c["A"].detach(), c["Bm"].detach(), c["Cm"].detach(), D=c["D"].detach(),
                           lengths=c["lengths"])
    before = _lib.launch_count()
    (dx,) = torch.autograd.grad((y, hT), c["x"], (gy.cuda(), gh.cuda()))
    assert _lib.launch_count() - before == 1 and torch.equal(dx, grads[0])


@pytest.mark.parametrize("B", [2, 9000])
def test_a_step_with_a_decay_of_minus_infinity(B):
    """Also where there are more sequences than threads."""
    from delrec.selective import selective_scan, selective_step
    d, _, _, _ = _inputs(1, B, 24, 8, torch.float32, None)
    d["A"][::3, ::2] = -float("inf")
    y, h = selective_step(d["x"][0], d["dt"][0], d["A"], d["Bm"][0], d["Cm"][0], d["h0"], D=d["D"], gate=d["gate"][0],
                          dt_bias=d["dt_bias"])
    ys, hs = selective_scan(d["x"], d["dt"], d["A"], d["Bm"], d["Cm"], d["h0"], D=d["D"], gate=d["gate"], dt_bias=d["dt_bias"])
    assert torch.isfinite(y).all() and torch.equal(h, hs)
    torch.testing.assert_close(y, ys[0], rtol=2.0 ** -18, atol=2.0 ** -18)     # the order of a sum of eight


@pytest.mark.parametrize("back", [False, True])
def test_growth_past_the_largest_number_of_a_state_that_is_zero(back):
    """A chunk of time may grow by more than a float holds; a state (or gradient) of 0 in front of it stays 0."""
    from delrec.selective import selective_scan
    T, N, S = 1024, 4, 4
    g = torch.Generator().manual_seed(8)
    rnd = lambda *s: torch.randn(*s, generator=g).cuda()   # noqa: E731
    dt, A = torch.ones(T, 1, N, device="cuda"), torch.full((N, S), 2.0, device="cuda")
    bm, cm, x = rnd(T, 1, S), rnd(T, 1, S), rnd(T, 1, N)
    gy = torch.ones(T, 1, N, device="cuda")
    if back:                               # only the first steps are looked at
        gy[10:] = 0
        x[10:] = 0
        bm[:] = 0
    else:
        x[:-10] = 0
    x.requires_grad_(True)
    y, hT = selective_scan(x, dt, A, bm, cm, softplus=False)
    (dx,) = torch.autograd.grad(y, x, gy)
    # the steps that matter alone, uncut
    part = slice(0, 10) if back else slice(T - 10, T)
    xs = x.detach()[part].clone().requires_grad_(True)
    ys, hs = selective_scan(xs, dt[part], A, bm[part], cm[part], softplus=False)
    (ds,) = torch.autograd.grad(ys, xs, gy[part])
    # (of steps that reach states a thousand steps on, e^2000 larger, dx is infinite by the formula, too)
    assert torch.isfinite(y).all() and torch.isfinite(dx[part]).all()
    # the sums cut in other places
    torch.testing.assert_close(y[part], ys, rtol=2.0 ** -18, atol=0)
    torch.testing.assert_close(dx[part], ds, rtol=2.0 ** -18, atol=0)
    if not back:
        torch.testing.assert_close(hT, hs, rtol=2.0 ** -18, atol=0)
        assert (y[:-10] == 0).all()


@pytest.mark.parametrize("B,N", [(4096, 8), (3001, 37)])
def test_parameter_gradients_are_rounded_once_over_sequences(B, N):
    """A sequence's sums for D and dt_bias are 8 + k 2^-20, exact in 24 bits; over the sequences they are added in 64."""
    from delrec.selective import selective_scan
    g = torch.Generator().manual_seed(0)
    x = torch.ones(8, B, N)
    x[0] += torch.randint(0, 1 << 19, (B, N), generator=g).float() * 2.0 ** -20
    xc = x.cuda()
    D, bias = torch.zeros(N, device="cuda", requires_grad=True), torch.zeros(N, device="cuda", requires_grad=True)
    A = torch.zeros(N, 1, device="cuda")
    ones = torch.ones(8, B, 1, device="cuda")
    last = torch.zeros(8, B, 1, device="cuda")
    last[7] = 1.0
    # without decay and with C = 1 at the last step alone, y_7 = sum of delta x + D x: d y_7 / d delta_t = x_t
    y, _ = selective_scan(xc, torch.zeros(8, B, N, device="cuda"), A, ones, last, D=D, dt_bias=bias, softplus=False)
    want = x.double().sum((0, 1)).float()
    assert torch.equal(torch.autograd.grad(y, D, torch.ones_like(y), retain_graph=True)[0].cpu(), want)
    gy = torch.zeros_like(y)
    gy[7] = 1.0
    assert torch.equal(torch.autograd.grad(y, bias, gy)[0].cpu(), want)
