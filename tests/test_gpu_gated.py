"""The gated linear recurrence (delrec.gated) against float64 loops over its formula: types,
gate groups, lengths, resets, strides, splits over time, single steps, 8-bit checkpoints.

Tolerances are the oracle's running bounds on fp32 arithmetic (16 units of 2^-24 of the
handled magnitudes per step) plus half a step of the stored type."""

import pytest
import torch

from oracle import sequence_oracle as O
from sequence_cases import within

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _inputs(T, B, N, D, dtype, seed=0, ragged=False, resets=False, h0=True, mean=2.0):
    g = torch.Generator().manual_seed(seed * 7919 + T * 31 + B * 17 + N + D)
    c = {"z": torch.randn(T, B, N, generator=g).to(dtype),
         "f": (torch.randn(T, B, N // D, generator=g) * 1.5 + mean).to(dtype),
         "h0": torch.randn(B, N, generator=g) if h0 else None,
         "gh": torch.randn(T, B, N, generator=g).to(dtype), "ghT": torch.randn(B, N, generator=g)}
    c["lengths"] = torch.randint(0, T + 1, (B,), generator=g) if ragged else None
    c["resets"] = torch.rand(T, B, generator=g) < 0.1 if resets else None
    return c


def _cuda(c):
    return {k: None if v is None else v.cuda() for k, v in c.items()}


def _check(c, decay_input=True, checkpoint8=False, lengths_dtype=torch.int32):
    from delrec.gated import gated_scan
    d = _cuda(c)
    z, f = d["z"].requires_grad_(True), d["f"].requires_grad_(True)
    h0 = d["h0"].requires_grad_(True) if d["h0"] is not None else None
    lens = d["lengths"].to(lengths_dtype) if d["lengths"] is not None else None
    h, hT = gated_scan(z, f, h0, lengths=lens, resets=d["resets"], decay_input=decay_input, checkpoint8=checkpoint8)
    leaves = [t for t in (z, f, h0) if t is not None]
    grads = torch.autograd.grad((h, hT), leaves, (d["gh"], d["ghT"]))
    kw = dict(lengths=c["lengths"], resets=c["resets"], decay_input=decay_input)
    r = O.gated_scan(c["z"], c["f"], c["h0"], **kw)
    within(h, r["h"], r["err"], "h")
    within(hT, r["hT"], r["errT"], "hT")
    bz, bf = c["z"].double(), c["f"].double()
    pre = r["pre"]
    perr = torch.zeros_like(pre)
    # the kept states' own bound, from the state after the step before
    perr[1:] = _carry(r["err"], c["lengths"])[:-1]
    if checkpoint8:
        bz, bf = O.restore8(bz), O.restore8(bf)
        states, e = O.recompute(bz, bf, pre, **kw)
        # a kept state's bound rides along inside its segment (gates are below 1)
        perr = e + perr[torch.arange(len(pre)) // 16 * 16]
        pre = states
    b = O.gated_scan_backward(bz, bf, pre, perr, c["gh"], c["ghT"], **kw)
    within(grads[0], b["dz"], b["ez"], "dz")
    within(grads[1], b["df"], b["ef"], "df")
    if h0 is not None:
        within(grads[2], b["dh0"], b["e0"], "dh0")
    return h, hT, grads


def _carry(err, lengths):
    """The bound of the state after each step (carried over padding)."""
    if lengths is None:
        return err
    out = err.clone()
    for t in range(1, err.shape[0]):
        past = t >= lengths
        out[t][past] = out[t - 1][past]
    return out


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,B,N", [(1, 1, 1), (1, 3, 40), (15, 2, 33), (16, 2, 32), (17, 1, 65), (40, 3, 31),
                                   (127, 2, 30), (128, 1, 64), (129, 2, 32), (300, 2, 7)])
def test_scan(T, B, N, dtype):
    _check(_inputs(T, B, N, 1, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,B,N", [(256, 1, 32), (600, 1, 40), (1024, 1, 32), (1100, 1, 3), (2111, 2, 33)])
def test_scan_split_over_a_cluster(T, B, N, dtype):
    """Few rows and long sequences: 2 to 8 blocks share a row's time."""
    _check(_inputs(T, B, N, 1, dtype, mean=4.0))


@pytest.mark.parametrize("decay_input", [True, False])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("D", [2, 3, 16, 20, 31, 32, 33, 64, 65, 130])
def test_scan_shared_gates(D, dtype, decay_input):
    _check(_inputs(37, 2, 3 * D, D, dtype), decay_input)


def test_scan_one_gate_for_all():
    _check(_inputs(140, 2, 257, 257, F32))


@pytest.mark.parametrize("lengths_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("T,D", [(20, 1), (20, 5), (200, 1), (700, 1), (200, 40)])
def test_scan_ragged(T, D, lengths_dtype):
    c = _inputs(T, 5, 2 * D if D > 1 else 34, D, F32, ragged=True, resets=True)
    c["lengths"][0], c["lengths"][1], c["lengths"][2] = 0, T, 1
    _check(c, lengths_dtype=lengths_dtype)
    _check(c, decay_input=False, lengths_dtype=lengths_dtype)


def test_padding_is_not_read_and_its_gradient_not_taken():
    c = _inputs(150, 4, 33, 1, F32, ragged=True)
    clean = _check(c)
    for k in ("z", "f", "gh"):
        for b in range(4):
            c[k][int(c["lengths"][b]):, b] = float("nan")
    c["z"][int(c["lengths"][0]):, 0] = float("inf")
    d = _cuda(c)
    from delrec.gated import gated_scan
    z, f, h0 = (d[k].requires_grad_(True) for k in ("z", "f", "h0"))
    h, hT = gated_scan(z, f, h0, lengths=d["lengths"])
    grads = torch.autograd.grad((h, hT), (z, f, h0), (d["gh"], d["ghT"]))
    for got, want in zip((h, hT, *grads), (clean[0], clean[1], *clean[2])):
        assert torch.equal(got, want)


def test_lengths_beyond_the_range_are_clamped():
    from delrec.gated import gated_scan
    c = _cuda(_inputs(20, 3, 8, 1, F32))
    a = gated_scan(c["z"], c["f"], c["h0"], lengths=torch.tensor([-5, 99, 20], device="cuda"))
    b = gated_scan(c["z"], c["f"], c["h0"], lengths=torch.tensor([0, 20, 20], device="cuda"))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("T", [30, 300, 1200])
def test_a_reset_drops_infinite_and_nan_states(T):
    """Sequences packed one after another: what diverged before a reset does not reach past it."""
    from delrec.gated import gated_scan
    c = _inputs(T, 1, 32, 1, F32, mean=0.0)
    cut = T - 7
    c["resets"] = torch.zeros(T, 1, dtype=torch.bool)
    c["resets"][cut] = True
    c["z"][2, :, :8] = float("inf")
    c["z"][T // 3, :, 8:16] = float("nan")
    d = _cuda(c)
    h, hT = gated_scan(d["z"], d["f"], d["h0"], resets=d["resets"])
    r = O.gated_scan(c["z"][cut:], c["f"][cut:], None)
    within(h[cut:], r["h"], r["err"], "h past the reset")
    within(hT, r["hT"], r["errT"], "hT")
    assert torch.isnan(h[T // 3:cut, :, 8:16]).all()


def test_packed_sequences_are_the_sequences_one_by_one():
    from delrec.gated import gated_scan
    c = _cuda(_inputs(90, 1, 48, 1, F32, h0=False))
    starts = [0, 13, 14, 61, 90]
    resets = torch.zeros(90, 1, dtype=torch.bool, device="cuda")
    resets[starts[:-1]] = True
    h, hT = gated_scan(c["z"], c["f"], resets=resets)
    for a, b in zip(starts, starts[1:]):
        one, last = gated_scan(c["z"][a:b], c["f"][a:b])
        torch.testing.assert_close(h[a:b], one, rtol=0, atol=2 ** -18)
    torch.testing.assert_close(hT, last, rtol=0, atol=2 ** -18)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), 100.0, -100.0, 90.0, -90.0])
def test_saturated_gates(value):
    c = _inputs(50, 2, 32, 1, F32)
    c["f"][10:14] = value
    c["f"][40, :, ::2] = value
    _check(c)
    _check(c, decay_input=False)


@pytest.mark.parametrize("T", [30, 200, 600])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(T, dtype):
    """Batch-major storage, channel slices, odd offsets, a gate expanded over time and rows, a
    strided channel dimension.  Alignment chooses how many channels a lane takes, and with it
    the order in which steps are put together: both orders are within 16 u per step of the
    exact value, carried on by gates below sigmoid(4.5) = 0.989, so within 2 * 16 u * 90 =
    2^-12.5 of each other times the largest magnitude (about 4 here: 2^-10.5), and 16-bit
    results within one step more."""
    from delrec.gated import gated_scan
    N, B = 32, 3
    g = torch.Generator().manual_seed(T)
    big = torch.randn(B, T, 3 * N + 1, generator=g).to(dtype).cuda()
    z, f = big[:, :, 1:N + 1].transpose(0, 1), big[:, :, N + 5:2 * N + 5].transpose(0, 1)
    gh = big[:, :, 2 * N:3 * N].transpose(0, 1)

    def go(z, f, gh):
        z, f = z.detach().requires_grad_(True), f.detach().requires_grad_(True)
        h, hT = gated_scan(z, f)
        return (h, hT, *torch.autograd.grad((h, hT), (z, f), (gh, torch.ones_like(hT))))

    def near(a, b):
        torch.testing.assert_close(a, b, rtol=2.0 ** -7 if a.dtype == BF16 else 0, atol=2.0 ** -10.5)

    base = go(z.contiguous(), f.contiguous(), gh.contiguous())
    channel_last = f.transpose(1, 2).contiguous().transpose(1, 2)
    for got in (go(z, f, gh), go(z.contiguous(), f, gh), go(z, channel_last, gh)):
        for a, b in zip(got, base):
            near(a, b)
    one = f[3:4, 1:2].expand(T, B, N)
    for a, b in zip(go(z, one, gh), go(z, one.contiguous(), gh)):
        near(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,B,N,D", [(1, 2, 33, 1), (45, 2, 40, 1), (150, 2, 64, 1), (520, 1, 32, 1),
                                     (45, 2, 60, 20), (33, 1, 200, 100)])
def test_checkpoint8(T, B, N, D, dtype):
    h, hT, _ = _check(_inputs(T, B, N, D, dtype), checkpoint8=True)
    from delrec.gated import gated_scan
    c = _cuda(_inputs(T, B, N, D, dtype))
    h1, hT1 = gated_scan(c["z"], c["f"], c["h0"])
    assert torch.equal(h, h1) and torch.equal(hT, hT1), "the forward pass does not depend on the checkpoint"


def test_checkpoint8_ragged():
    c = _inputs(130, 5, 40, 1, F32, ragged=True, resets=True)
    c["lengths"][0] = 0
    _check(c, checkpoint8=True)
    _check(c, decay_input=False, checkpoint8=True)


def test_gradients_by_differences():
    """d loss along random directions of z, f, h0 against central differences of the float64 loop."""
    from delrec.gated import gated_scan
    c = _inputs(60, 2, 24, 3, F32, resets=True)
    d = _cuda(c)
    z, f, h0 = (d[k].requires_grad_(True) for k in ("z", "f", "h0"))
    h, hT = gated_scan(z, f, h0, resets=d["resets"])
    grads = torch.autograd.grad((h, hT), (z, f, h0), (d["gh"], d["ghT"]))
    g = torch.Generator().manual_seed(1)

    def loss(z, f, h0):
        r = O.gated_scan(z, f, h0, resets=c["resets"])
        return (r["h"] * c["gh"].double()).sum() + (r["hT"] * c["ghT"].double()).sum()

    eps = 1e-5
    base = [c[k].double() for k in ("z", "f", "h0")]
    for i, grad in enumerate(grads):
        v = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + eps * v, base[i] - eps * v
        num = (loss(*up) - loss(*dn)) / (2 * eps)
        ana = (grad.double().cpu() * v).sum()
        # central differences: eps^2 |third derivative| + 2^-53 |loss| / eps; fp32 gradients: 2^-18
        scale = (grad.double().cpu() * v).abs().sum()
        assert abs(num - ana) < 1e-5 * scale


def test_partial_gradients():
    from delrec.gated import gated_scan
    c = _cuda(_inputs(40, 2, 33, 1, F32))
    full = None
    for only in (None, "z", "f", "h0"):
        t = {k: c[k].detach().requires_grad_(only in (None, k)) for k in ("z", "f", "h0")}
        h, hT = gated_scan(t["z"], t["f"], t["h0"])
        leaves = [t[k] for k in ("z", "f", "h0") if only in (None, k)]
        got = torch.autograd.grad((h, hT), leaves, (c["gh"], c["ghT"]))
        if only is None:
            full = dict(zip(("z", "f", "h0"), got))
        else:
            assert torch.equal(got[0], full[only])
    t = {k: c[k].detach().requires_grad_(True) for k in ("z", "f", "h0")}
    h, hT = gated_scan(t["z"], t["f"], t["h0"])
    a = torch.autograd.grad(hT, list(t.values()), c["ghT"], retain_graph=True)
    b = torch.autograd.grad(h, list(t.values()), c["gh"], retain_graph=True)
    for x, y, w in zip(a, b, full.values()):
        torch.testing.assert_close(x + y, w, rtol=2 ** -18, atol=2 ** -18)
    again = torch.autograd.grad((h, hT), list(t.values()), (c["gh"], c["ghT"]))
    for x, w in zip(again, full.values()):
        assert torch.equal(x, w)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,N,D", [(1, 1, 1), (5, 33, 1), (64, 512, 1), (3, 60, 20), (2, 130, 65)])
def test_step(B, N, D, dtype):
    from delrec.gated import gated_step
    c = _inputs(1, B, N, D, dtype)
    d = _cuda(c)
    for di in (True, False):
        h, nxt = gated_step(d["z"][0], d["f"][0], d["h0"], decay_input=di)
        r = O.gated_scan(c["z"], c["f"], c["h0"], decay_input=di)
        within(h, r["h"][0], r["err"][0], "h")
        within(nxt, r["hT"], r["errT"], "next")
        state = d["h0"].clone()
        h2, same = gated_step(d["z"][0], d["f"][0], state, decay_input=di, out=state)
        assert same is state and torch.equal(state, nxt) and torch.equal(h2, h)
    h, nxt = gated_step(d["z"][0], d["f"][0])
    r = O.gated_scan(c["z"], c["f"], None)
    within(nxt, r["hT"], r["errT"], "next from nothing")
    active = torch.arange(B, device="cuda") % 2 == 1
    z = d["z"][0].clone()
    z[~active] = float("nan")
    h, nxt = gated_step(z, d["f"][0], d["h0"], active=active)
    assert torch.equal(nxt[~active], d["h0"][~active]) and not h[~active].any() and torch.isfinite(nxt).all()


def test_steps_are_the_scan():
    from delrec.gated import gated_scan, gated_step
    c = _cuda(_inputs(37, 4, 70, 7, F32))
    h, hT = gated_scan(c["z"], c["f"], c["h0"])
    state = c["h0"].clone()
    for t in range(37):
        one, _ = gated_step(c["z"][t], c["f"][t], state, out=state)
        torch.testing.assert_close(one, h[t], rtol=2 ** -19, atol=2 ** -19)
    torch.testing.assert_close(state, hT, rtol=2 ** -19, atol=2 ** -19)


@pytest.mark.parametrize("shape", [(0, 2, 5), (4, 0, 5), (4, 2, 0)])
def test_empty(shape):
    from delrec.gated import gated_scan
    T, B, N = shape
    z = torch.randn(T, B, N, device="cuda", requires_grad=True)
    f = torch.randn(T, B, N, device="cuda", requires_grad=True)
    h0 = torch.randn(B, N, device="cuda", requires_grad=True)
    h, hT = gated_scan(z, f, h0)
    assert h.shape == shape and torch.equal(hT, h0)
    g = torch.autograd.grad((h, hT), (z, f, h0), (torch.ones_like(h), torch.ones_like(hT)))
    assert torch.equal(g[2], torch.ones_like(h0))


def test_same_bits_every_time_and_on_other_streams():
    from delrec.gated import gated_scan
    c = _cuda(_inputs(900, 2, 64, 1, F32))

    def go():
        z, f = c["z"].detach().requires_grad_(True), c["f"].detach().requires_grad_(True)
        h, hT = gated_scan(z, f, c["h0"])
        return (h, hT, *torch.autograd.grad((h, hT), (z, f), (c["gh"], c["ghT"])))

    base = go()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(s):
            other = go()
        torch.cuda.current_stream().wait_stream(s)
        for a, b in zip(other, base):
            assert torch.equal(a, b)


def test_captured_in_a_graph():
    """Training pass and step in two captured graphs, replayed with new inputs, one after the other
    and interleaved."""
    from delrec.gated import gated_scan, gated_step
    c = _cuda(_inputs(300, 2, 80, 40, F32))

    def train():
        z, f = c["z"].detach().requires_grad_(True), c["f"].detach().requires_grad_(True)
        h, hT = gated_scan(z, f, c["h0"])
        return (h.detach(), hT.detach(), *torch.autograd.grad((h, hT), (z, f), (c["gh"], c["ghT"])))

    def step():
        return gated_step(c["z"][0], c["f"][0], c["h0"])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        train(), step()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for fn in (train, step, train):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(fn())
        graphs.append(g)
    for seed in (1, 2):
        for k, v in _cuda(_inputs(300, 2, 80, 40, F32, seed=seed)).items():
            if v is not None:
                c[k].copy_(v)
        for g in graphs:
            g.replay()
        want = [train(), step(), train()]
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            for a, b in zip(got, ref):
                assert torch.equal(a, b)


def test_many_rows():
    """More rows than blocks fit at once, one segment and several."""
    for T in (5, 140):
        c = _inputs(T, 1, 32, 1, F32)
        reps = 3000
        d = {k: (v.repeat(*([1, reps, 1] if v.dim() == 3 else [reps, 1])).cuda() if v is not None else None)
             for k, v in c.items()}
        from delrec.gated import gated_scan
        z, f = d["z"].requires_grad_(True), d["f"].requires_grad_(True)
        h, hT = gated_scan(z, f, d["h0"])
        dz, df = torch.autograd.grad((h, hT), (z, f), (d["gh"], d["ghT"]))
        for t in (h, dz, df):
            assert torch.equal(t, t[:, :1].expand_as(t))
        r = O.gated_scan(c["z"], c["f"], c["h0"])
        within(h[:, :1], r["h"], r["err"], "h")
