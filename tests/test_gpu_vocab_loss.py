"""The vocabulary losses against their formulas in float64."""

import pytest
import torch

from sequence_cases import FLOOR, HALF, within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24

# T, B, D, V, bias, reduction, lengths
CASES = [(1, 1, 1, 1, False, "mean", None), (1, 3, 8, 5, True, "none", None), (3, 5, 40, 129, True, "mean", [3, 0, 1, 3, 2]),
         (7, 20, 64, 1000, False, "sum", None), (5, 30, 33, 700, True, "none", None), (2, 129, 136, 257, False, "mean", None),
         (9, 33, 130, 3001, True, "mean", list(range(9)) * 3 + [9] * 6), (3, 64, 264, 515, False, "none", None)]


def _make(case, dtype, K=0, seed=0, scale=2.0):
    T, B, D, V, bias, reduction, lengths = case
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    d = dict(x=rnd(T, B, D).to(dtype), w=(rnd(V, D) * scale * D ** -0.5).to(dtype), bias=rnd(V).to(dtype) if bias else None,
             reduction=reduction, lengths=torch.tensor(lengths) if lengths else None)
    if K:
        d["index"] = torch.randint(0, V, (T, B, K), generator=g)
        d["logits"] = rnd(T, B, K) * 2
        # entries left out, one way or the other, and positions that keep nothing
        d["index"][torch.rand(T, B, K, generator=g) < 0.1] = -1
        d["logits"][torch.rand(T, B, K, generator=g) < 0.1] = -float("inf")
        d["index"][torch.rand(T, B, generator=g) < 0.1] = -7
    else:
        d["index"] = torch.randint(0, V, (T, B), generator=g)
        d["index"][torch.rand(T, B, generator=g) < 0.2] = -100
    grad = rnd(T, B) if reduction == "none" else torch.tensor(1.7)
    return d, grad


def _call(c, tau=1.0, **kw):
    from delrec.vocab_loss import linear_cross_entropy, linear_distill
    if c.get("logits") is None:
        return linear_cross_entropy(c["x"], c["w"], c["index"], c["bias"], reduction=c["reduction"], lengths=c["lengths"], **kw)
    return linear_distill(c["x"], c["w"], c["index"], c["logits"], c["bias"], temperature=tau, reduction=c["reduction"],
                          lengths=c["lengths"], **kw)


def _cuda(d):
    return {k: v.cuda() if torch.is_tensor(v) else v for k, v in d.items()}


def _compare(d, grad, dtype, tau=1.0):
    from oracle import selective_oracle as O
    ref = O.vocab_loss(**d, tau=tau, g=grad, half=HALF[dtype] if dtype != torch.float32 else 4 * U)
    c = _cuda(d)
    if c["lengths"] is not None:           # what stands past a length is not read
        past = torch.arange(d["x"].shape[0], device="cuda")[:, None] >= c["lengths"][None]
        c["x"] = torch.where(past.unsqueeze(-1), torch.full_like(c["x"], float("nan")), c["x"])
        m = past if c.get("logits") is None else past.unsqueeze(-1)
        c["index"] = torch.where(m, torch.full_like(c["index"], 1 << 40), c["index"])
    if c.get("logits") is None:            # nor x at a position that does not count
        c["x"] = torch.where((c["index"] == -100).unsqueeze(-1), torch.full_like(c["x"], float("inf")), c["x"])
    leaves = [k for k in ("x", "w", "bias") if c[k] is not None]
    for k in leaves:
        c[k].requires_grad_(True)
    loss = _call(c, tau)
    within(loss, ref["loss"], ref["e_loss"], "loss")
    grads = torch.autograd.grad(loss, [c[k] for k in leaves], grad.cuda())
    for k, v in zip(leaves, grads):
        name = {"x": "dx", "w": "dw", "bias": "db"}[k]
        within(v, ref[name], ref["e_" + name], name)
    with torch.no_grad():
        assert torch.equal(_call(c, tau), loss)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_cross_entropy_against_float64(case, dtype):
    _compare(*_make(case, dtype), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,tau", [(1, 1.0), (5, 2.0), (33, 1.0), (130, 0.5)])
@pytest.mark.parametrize("case", [CASES[2], CASES[4], CASES[5]])
def test_distillation_against_float64(case, K, tau, dtype):
    """Lists with repeated indices, entries and whole positions left out."""
    _compare(*_make(case, dtype, K), dtype, tau)


@pytest.mark.parametrize("teacher", DTYPES)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_types_of_a_teacher(teacher, index):
    d, grad = _make(CASES[3], torch.bfloat16, 9)
    d["logits"], d["index"] = d["logits"].to(teacher), d["index"].to(index)
    _compare(d, grad, torch.bfloat16, 2.0)


def test_several_pieces_of_the_vocabulary(monkeypatch):
    """More positions than the logits' gradient has room for at once."""
    d, grad = _make((128, 400, 16, 2600, True, "mean", None), torch.bfloat16)
    c = _cuda(d)
    for k in ("x", "w", "bias"):
        c[k].requires_grad_(True)
    loss = _call(c)
    got = torch.autograd.grad(loss, [c["x"], c["w"], c["bias"]], grad.cuda())
    x, w, b = (c[k].detach().double().requires_grad_(True) for k in ("x", "w", "bias"))
    ref = torch.nn.functional.cross_entropy((x @ w.t() + b).flatten(0, 1), c["index"].flatten(), ignore_index=-100)
    # 51200 positions: a mean of losses good to (D / 16 + 12) 2 u of the logits' magnitudes (below 20) and 150 u each
    assert abs(loss.item() - ref.item()) <= U * (26 * 20 + 150 + 8 * ref.item())
    want = torch.autograd.grad(ref, [x, w, b], grad.cuda().double())
    n = (c["index"] != -100).sum().item()
    for got1, want1, k in zip(got, want, "xwb"):
        # each entry of G is rounded once: at most 2^-8 of sum |G| |operand| (|operand| < 6) and the result's rounding;
        # sum over the vocabulary of |G| is at most 2 / n, over the positions at most twice the column's share
        d64 = (got1.double() - want1).abs()
        if k == "x":
            assert (d64 <= 2.0 ** -8 * (1.7 * 2 / n * 6 + want1.abs()) * 1.01).all()
        else:
            q = torch.softmax((x @ w.t() + b).detach().flatten(0, 1), 1)
            q = q * (c["index"].flatten() != -100).unsqueeze(1)
            share = q.sum(0) + torch.bincount(c["index"].flatten()[c["index"].flatten() >= 0], minlength=2600)
            bound = 2.0 ** -8 * (1.7 / n * share * 6)
            assert (d64 <= (bound.unsqueeze(1) if k == "w" else bound) + 2.0 ** -8 * want1.abs() * 1.01).all()


def test_gradient_against_differences():
    """The float64 oracle's gradients are those of its own forward pass."""
    from oracle import selective_oracle as O
    for K, tau in ((0, 1.0), (4, 2.0)):
        d, grad = _make((3, 4, 6, 11, True, "none", None), torch.float32, K, 2)
        d = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in d.items()}
        grad = grad.double()
        ref = O.vocab_loss(**d, tau=tau, g=grad)
        value = lambda e: (O.vocab_loss(**e, tau=tau)["loss"] * grad).sum()   # noqa: E731
        for k, name in (("x", "dx"), ("w", "dw"), ("bias", "db")):
            v = torch.randn(d[k].shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
            diff = (value({**d, k: d[k] + 1e-5 * v}) - value({**d, k: d[k] - 1e-5 * v})) / 2e-5
            assert abs(diff - (ref[name] * v).sum()) <= 1e-7 * (1 + (ref[name] * v).abs().sum()), name


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("K", [0, 3])
def test_nothing_counts(K, reduction):
    d, grad = _make((4, 6, 24, 50, True, reduction, None), torch.bfloat16, K)
    d["index"].fill_(-100)
    c = _cuda(d)
    for k in ("x", "w", "bias"):
        c[k].requires_grad_(True)
    loss = _call(c)
    assert not loss.any() and loss.shape == ((4, 6) if reduction == "none" else ())
    for v in torch.autograd.grad(loss, [c[k] for k in ("x", "w", "bias")], grad.cuda()):
        assert not v.any()


def test_indices_past_the_vocabulary_are_not_read():
    """Their losses are NaN, the status word says so, the other positions' losses are as they were."""
    from delrec import _lib
    for K in (0, 4):
        d, _ = _make((2, 40, 32, 60, False, "none", None), torch.float32, K)
        c = _cuda(d)
        want = _call(c)
        bad = c["index"].clone()
        flat = bad.view(80, -1)
        flat[3, 0], flat[50, -1] = 60, 1 << 40
        if not K:
            flat[7, 0] = -1
        if K:
            c["logits"][0, 3] = c["logits"][1, 10] = 0.0
            want = _call(c)
        assert _lib.status() == 0
        got = _call({**c, "index": bad})
        assert _lib.status() & 2
        _lib.check(_lib.lib().delrec_clear_status(), "clear")
        rows = [3, 50] + ([] if K else [7])
        assert got.flatten()[rows].isnan().all()
        keep = torch.ones(80, dtype=torch.bool, device="cuda")
        keep[rows] = False
        assert torch.equal(got.flatten()[keep], want.flatten()[keep])
        c["x"].requires_grad_(True)
        loss = _call({**c, "index": bad})
        dx, = torch.autograd.grad(loss, c["x"], torch.ones_like(loss))
        dx = dx.view(80, -1)
        assert dx[rows].isnan().all() and torch.isfinite(dx[keep]).all()
        _lib.check(_lib.lib().delrec_clear_status(), "clear")


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_logits_and_tiny_gradients(dtype):
    """Logits far apart and gradients far below the type's smallest value: the scale is a power of two."""
    d, grad = _make((4, 30, 32, 200, False, "none", None), dtype, scale=40.0)
    _compare(d, grad, dtype)
    d, grad = _make((4, 30, 32, 200, False, "none", None), dtype)
    c = _cuda(d)
    c["w"].requires_grad_(True)
    one, = torch.autograd.grad(_call(c), c["w"], grad.cuda())
    small, = torch.autograd.grad(_call(c), c["w"], grad.cuda() * 2.0 ** -10)
    # one power of two scales both, so their sums are the same; `one` is off by half a step of its own, and
    # `small` by half a step of its own, in fp16 down to 2^-25
    want = one.double() * 2.0 ** -10
    step = HALF[dtype] * want.abs()
    assert ((small.double() - want).abs() <= step + torch.maximum(step, torch.full_like(step, FLOOR[dtype]))).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Strided and odd-addressed tensors, and other leading shapes, give the same numbers."""
    d, grad = _make((6, 10, 40, 300, True, "none", None), dtype)
    c = _cuda(d)
    grad = grad.cuda()

    def go(x=c["x"], w=c["w"], index=c["index"], g=grad):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = _call({**c, "x": x, "w": w, "index": index})
        return [loss, *torch.autograd.grad(loss, (x, w), g)]

    want = go()
    forms = [lambda v: v.transpose(0, 1).contiguous().transpose(0, 1), lambda v: torch.stack([v, v], -1)[..., 0],
             lambda v: torch.cat([v.new_zeros(1), v.flatten()])[1:].view(v.shape)]
    for form in forms:
        for got in (go(x=form(c["x"])), go(w=form(c["w"])), go(index=form(c["index"]), g=form(grad))):
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    for shape in ((60,), (2, 3, 10)):
        got = go(x=c["x"].view(*shape, 40), index=c["index"].view(shape), g=grad.view(shape))
        assert got[0].shape == shape
        for a, b in zip(got, want):
            assert torch.equal(a, b.view(a.shape))


def test_no_positions():
    from delrec.vocab_loss import linear_cross_entropy
    w = torch.randn(9, 4, device="cuda", requires_grad=True)
    for shape in ((0, 3), (3, 0), (0,)):
        x = torch.randn(*shape, 4, device="cuda", requires_grad=True)
        t = torch.zeros(shape, dtype=torch.int64, device="cuda")
        loss = linear_cross_entropy(x, w, t)
        dx, dw = torch.autograd.grad(loss, (x, w))
        assert loss.item() == 0 and dx.shape == x.shape and not dw.any()
        assert linear_cross_entropy(x, w, t, reduction="none").shape == shape


@pytest.mark.parametrize("teacher", DTYPES)
def test_teacher_logits_of_the_lowest_value(teacher):
    """A mask of the type's lowest value keeps its entries: next to others they weigh nothing, alone they
    weigh the same, and no temperature makes them infinite.  The same bits as with logits that mean it."""
    d, grad = _make((3, 7, 24, 50, True, "none", None), torch.float32, 5, seed=11)
    d["index"] = d["index"].clamp(min=0)
    plain = torch.randn(3, 7, 5, generator=torch.Generator().manual_seed(3)).to(teacher)
    plain[0, :, 1:4] = -1e4                # exp(-1e4 / 3) is 0
    plain[1] = 0
    lowest = plain.clone()
    lowest[0, :, 1:4] = torch.finfo(teacher).min
    lowest[1] = torch.finfo(teacher).min
    for tau in (0.25, 1.0, 3.0):
        out = []
        for logits in (plain, lowest):
            c = _cuda(dict(d, logits=logits))
            leaves = [c[k].requires_grad_(True) for k in ("x", "w", "bias")]
            loss = _call(c, tau)
            out.append([loss] + list(torch.autograd.grad(loss, leaves, grad.cuda())))
        assert all(torch.isfinite(v).all() for v in out[0])
        assert all(torch.equal(u, v) for u, v in zip(*out))


def test_many_positions():
    """More positions than the packing counts by itself: the same bits as in two calls."""
    from delrec.vocab_loss import linear_cross_entropy
    g = torch.Generator().manual_seed(5)
    M = 140001
    x = torch.randn(M, 16, generator=g).to("cuda", torch.bfloat16).requires_grad_(True)
    w = torch.randn(24, 16, generator=g).to("cuda", torch.bfloat16)
    t = torch.randint(0, 24, (M,), generator=g)
    t[torch.rand(M, generator=g) < 0.3] = -100
    t[4096:9000] = -100
    t = t.cuda()
    loss = linear_cross_entropy(x, w, t, reduction="none")
    dx, = torch.autograd.grad(loss, x, torch.ones_like(loss))
    for part in (slice(0, 60000), slice(60000, 120000), slice(120000, M)):
        y = x.detach()[part].clone().requires_grad_(True)
        l = linear_cross_entropy(y, w, t[part], reduction="none")
        assert torch.equal(l, loss[part])
        assert torch.equal(torch.autograd.grad(l, y, torch.ones_like(l))[0], dx[part])
    assert (dx[t == -100] == 0).all() and (loss[t == -100] == 0).all() and (loss[t >= 0] > 0).all()
