"""The short causal convolution against its formula in float64."""

import pytest
import torch

from sequence_cases import within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]

# T, B, N, K, act, bias, state, lengths, resets
CASES = [(1, 1, 1, 1, "silu", True, False, None, False), (1, 3, 8, 4, "silu", True, True, None, False),
         (2, 2, 5, 8, "none", False, True, None, True), (37, 3, 40, 4, "silu", True, True, [0, 37, 2], True),
         (130, 2, 16, 3, "silu", False, False, [130, 61], False), (131, 2, 7, 2, "none", True, True, [1, 130], True),
         (200, 1, 12, 8, "silu", True, True, None, True), (64, 4, 24, 5, "silu", True, True, [64, 3, 0, 65], True),
         (50, 2, 36, 6, "none", False, False, None, False), (19, 2, 130, 7, "silu", True, True, [7, 19], True)]


def _make(case, dtype, seed=0):
    T, B, N, K, act, bias, state, lengths, resets = case
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    d = dict(x=rnd(T, B, N).to(dtype), w=rnd(N, K) * K ** -0.5, b=rnd(N) if bias else None,
             state=rnd(K - 1, B, N).to(dtype) if state else None, act=act,
             lengths=torch.tensor(lengths) if lengths else None,
             resets=torch.rand(T, B, generator=g) < 0.2 if resets else None)
    return d, rnd(T, B, N).to(dtype), rnd(K - 1, B, N).to(dtype)


def _cuda(v):
    return v.cuda() if torch.is_tensor(v) else v


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_against_float64(case, dtype):
    from delrec.short_conv import short_conv
    from oracle import selective_oracle as O
    d, gy, gs = _make(case, dtype)
    ref = O.short_conv(**d, gy=gy, gs=gs)
    c = {k: _cuda(v) for k, v in d.items()}
    if c["lengths"] is not None:           # what stands past a length is not read
        past = torch.arange(case[0], device="cuda")[:, None] >= c["lengths"][None]
        c["x"] = torch.where(past.unsqueeze(-1), torch.full_like(c["x"], float("nan")), c["x"])
        gy = torch.where(past.cpu().unsqueeze(-1), torch.full_like(gy, float("inf")), gy)
    leaves = [k for k in ("x", "w", "b", "state") if c[k] is not None]
    for k in leaves:
        c[k].requires_grad_(True)
    y, new = short_conv(c["x"], c["w"], c["b"], c["state"], act=c["act"], lengths=c["lengths"], resets=c["resets"])
    within(y, ref["y"], ref["e_y"], "y")
    within(new, ref["new"], ref["e_new"], "new state")
    grads = torch.autograd.grad((y, new), [c[k] for k in leaves], (gy.cuda(), gs.cuda()))
    for k, v in zip(leaves, grads):
        name = {"x": "dx", "w": "dw", "b": "db", "state": "ds"}[k]
        within(v, ref[name], ref["e_" + name], name)
    with torch.no_grad():                   # the same bits without a backward pass
        y2, new2 = short_conv(c["x"], c["w"], c["b"], c["state"], act=c["act"], lengths=c["lengths"], resets=c["resets"])
    assert torch.equal(y, y2) and torch.equal(new, new2)


def test_gradient_against_differences():
    """The float64 oracle's gradients are those of its own forward pass."""
    from oracle import selective_oracle as O
    d, gy, gs = _make((9, 2, 3, 3, "silu", True, True, [9, 4], True), torch.float32, 5)
    d = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in d.items()}
    gy, gs = gy.double(), gs.double()
    ref = O.short_conv(**d, gy=gy, gs=gs)
    value = lambda e: (lambda r: (r["y"] * gy).sum() + (r["new"] * gs).sum())(O.short_conv(**e))   # noqa: E731
    for k, name in (("x", "dx"), ("w", "dw"), ("b", "db"), ("state", "ds")):
        v = torch.randn(d[k].shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
        if k == "x":
            v[4:, 1] = 0
        diff = (value({**d, k: d[k] + 1e-5 * v}) - value({**d, k: d[k] - 1e-5 * v})) / 2e-5
        assert abs(diff - (ref[name] * v).sum()) <= 1e-7 * (1 + (ref[name] * v).abs().sum()), name


@pytest.mark.parametrize("dtype", DTYPES)
def test_pieces_and_steps_give_the_whole(dtype):
    """A sequence in pieces, and in single steps with the state updated in place, has the whole one's bits."""
    from delrec.short_conv import short_conv, short_conv_step
    d, _, _ = _make((23, 3, 20, 4, "silu", True, True, None, False), dtype)
    c = {k: _cuda(v) for k, v in d.items()}
    y, new = short_conv(c["x"], c["w"], c["b"], c["state"])
    y1, s = short_conv(c["x"][:2], c["w"], c["b"], c["state"])
    y2, s = short_conv(c["x"][2:], c["w"], c["b"], s)
    assert torch.equal(torch.cat([y1, y2]), y) and torch.equal(s, new)
    s = c["state"].clone()
    for t in range(23):
        yt, out = short_conv_step(c["x"][t], c["w"], c["b"], s, out=s)
        assert out is s and torch.equal(yt, y[t])
    assert torch.equal(s, new)
    # rows that are not active keep their state
    active = torch.tensor([True, False, True], device="cuda")
    before = s.clone()
    yt, nxt = short_conv_step(c["x"][0], c["w"], c["b"], s, active=active)
    full, moved = short_conv_step(c["x"][0], c["w"], c["b"], s)
    assert torch.equal(nxt[:, 1], before[:, 1]) and not yt[1].any() and torch.equal(s, before)
    assert torch.equal(nxt[:, [0, 2]], moved[:, [0, 2]]) and torch.equal(yt[[0, 2]], full[[0, 2]])
    assert torch.equal(short_conv_step(c["x"][0], c["w"], c["b"])[0], short_conv(c["x"][:1], c["w"], c["b"])[0][0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Batch-major tensors, strided channels and odd addresses give the same numbers."""
    from delrec.short_conv import short_conv
    d, gy, gs = _make((40, 3, 24, 4, "silu", True, True, None, False), dtype)
    c = {k: _cuda(v) for k, v in d.items()}
    gy, gs = gy.cuda(), gs.cuda()

    def go(x, w=c["w"], state=c["state"], gy=gy):
        x = x.requires_grad_(True)
        y, new = short_conv(x, w, c["b"], state)
        return [y, new, *torch.autograd.grad((y, new), (x,), (gy, gs))]

    want = go(c["x"].clone())
    forms = [lambda v: v.transpose(0, 1).contiguous().transpose(0, 1).detach(),
             lambda v: torch.stack([v, v], -1).detach()[..., 0],
             lambda v: torch.cat([v.new_zeros(1), v.flatten()]).detach()[1:].view(v.shape)]
    for form in forms:
        for a, b in zip(go(form(c["x"])), want):
            assert torch.equal(a, b)
        for a, b in zip(go(c["x"].clone(), gy=form(gy)), want):
            assert torch.equal(a, b)
    for a, b in zip(go(c["x"].clone(), state=forms[2](c["state"]), w=forms[1](c["w"])), want):
        assert torch.equal(a, b)


def test_empty_sequences():
    from delrec.short_conv import short_conv
    w, b = torch.randn(6, 3, device="cuda", requires_grad=True), torch.randn(6, device="cuda", requires_grad=True)
    for shape in ((0, 2, 6), (4, 0, 6)):
        x = torch.randn(shape, device="cuda", requires_grad=True)
        state = torch.randn(2, shape[1], 6, device="cuda", requires_grad=True)
        y, new = short_conv(x, w, b, state)
        assert y.shape == x.shape and torch.equal(new, state)
        grads = torch.autograd.grad((y, new), (x, w, b, state), (torch.ones_like(y), torch.full_like(new, 2.0)))
        assert grads[0].shape == x.shape and not grads[1].any() and not grads[2].any()
        assert torch.equal(grads[3], torch.full_like(state, 2.0))


def test_one_of_two_gradients():
    """Only y, or only the new state, is used."""
    from delrec.short_conv import short_conv
    from oracle import selective_oracle as O
    d, gy, gs = _make((11, 2, 6, 4, "silu", True, True, None, False), torch.float32)
    for use in ("y", "new"):
        c = {k: _cuda(v) for k, v in d.items()}
        c["x"].requires_grad_(True)
        y, new = short_conv(c["x"], c["w"], c["b"], c["state"])
        ref = O.short_conv(**d, **(dict(gy=gy) if use == "y" else dict(gs=gs)))
        (dx,) = torch.autograd.grad(y if use == "y" else new, c["x"], (gy if use == "y" else gs).cuda())
        within(dx, ref["dx"], ref["e_dx"], "dx")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", range(1, 9))
@pytest.mark.parametrize("N", [5, 12])
def test_steps_of_every_filter(dtype, K, N):
    """Two single steps have the bits of a walk over two rows, wherever the filter stands in memory."""
    from delrec.short_conv import short_conv, short_conv_step
    g = torch.Generator().manual_seed(K)
    B = 7
    x = torch.randn(2, B, N, generator=g).to("cuda", dtype)
    w = torch.randn(N * K + 1, generator=g).cuda()[1:].view(N, K)
    b = torch.randn(N, generator=g).cuda()
    s = torch.randn(K - 1, B, N, generator=g).to("cuda", dtype)
    want, last = short_conv(x, w, b, s)
    for filt in (w, w.clone()):
        out = s.clone()
        for t in range(2):
            y, out = short_conv_step(x[t], filt, b, out, out=out)
            assert torch.equal(y, want[t])
        assert torch.equal(out, last)
