"""Tokens masked through the bias, by -inf or by the type's lowest value, and temperatures at their limits."""

import pytest
import torch

from sequence_cases import HALF

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(dtype, M=70, D=48, V=300, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, D, generator=g).to("cuda", dtype).requires_grad_(True)
    w = (torch.randn(V, D, generator=g) * 2 * D ** -0.5).to("cuda", dtype).requires_grad_(True)
    b = torch.randn(V, generator=g).to("cuda", dtype)
    dead = (torch.rand(V, generator=g) < 0.3).cuda()
    dead[:2] = True
    live = (~dead).nonzero()[:, 0]
    t = live[torch.randint(0, live.numel(), (M,), generator=g).cuda()]
    return x, w, b, dead, live, t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lowest", [False, True])
def test_masked_tokens(lowest, dtype):
    """A masked token takes no part: the losses are those without it, its rows of the gradients are 0."""
    from delrec.vocab_loss import linear_cross_entropy, linear_distill
    x, w, b, dead, live, t = _inputs(dtype)
    bias = torch.where(dead, torch.full_like(b, torch.finfo(dtype).min if lowest else -float("inf")), b).requires_grad_(True)
    idx = torch.stack([t, live[torch.arange(70, device="cuda") % live.numel()]], 1)
    logits = torch.randn(70, 2, generator=torch.Generator().manual_seed(1)).cuda()
    z = (x.detach().double() @ w.detach()[live].double().t() + b[live].double())
    p = torch.softmax(logits.double() / 2, 1)
    pos = torch.searchsorted(live, idx)
    for K in (0, 2):
        if K:
            loss = linear_distill(x, w, idx, logits, bias, temperature=2.0, reduction="none")
            want = 4 * (p * (p.log() - torch.log_softmax(z / 2, 1).gather(1, pos))).sum(1)
        else:
            loss = linear_cross_entropy(x, w, t, bias, reduction="none")
            want = torch.nn.functional.cross_entropy(z, pos[:, 0], reduction="none")
        # logits of magnitudes below 30, (D / 16 + 12) 2 u of them twice; exponents, sums and p 300 u; tau^2
        assert ((loss.double() - want).abs() <= (4 if K else 1) * U * (30 * 30 * 2 + 300)).all()
        dx, dw, db = torch.autograd.grad(loss, (x, w, bias), torch.ones_like(loss))
        assert (dw[dead] == 0).all() and (db[dead] == 0).all()
        assert all(torch.isfinite(v).all() for v in (dx, dw, db))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [0, 1, 3])
def test_a_masked_target(K, dtype):
    """-inf there makes the loss infinite, the type's lowest value the number that it is; the gradients are finite, q = 0."""
    from delrec.vocab_loss import linear_cross_entropy, linear_distill
    x, w, b, dead, live, t = _inputs(dtype, seed=2)
    t = t.clone()
    t[5] = 0
    for low in (-float("inf"), torch.finfo(dtype).min):
        bias = torch.where(dead, torch.full_like(b, low), b).requires_grad_(True)
        if K:
            idx = torch.stack([t] + [live[:70]] * (K - 1), 1)
            loss = linear_distill(x, w, idx, torch.zeros(70, K, device="cuda"), bias, reduction="none")
        else:
            loss = linear_cross_entropy(x, w, t, bias, reduction="none")
        others = torch.arange(70, device="cuda") != 5
        assert torch.isfinite(loss[others]).all()
        want = -low / max(K, 1)
        if low == -float("inf"):
            assert loss[5] == want
        else:
            # other terms are below 100; 8 u of the value itself
            assert abs(loss[5].item() - want) <= 100 + 8 * U * want
        grads = torch.autograd.grad(loss, (x, w, bias), torch.ones_like(loss))
        assert all(torch.isfinite(v).all() for v in grads)
        # the position's share of its target is all that reaches bias[0]: q - p = -1 / K there
        assert abs(grads[2][0].item() + 1 / max(K, 1)) <= HALF[dtype] + 4 * U


def test_temperatures_at_their_limits():
    """From 1e-6 to 1e6, against float64; past those refused."""
    from delrec.vocab_loss import linear_distill
    x, w, b, _, live, t = _inputs(torch.float32)
    logits = torch.randn(70, 3, generator=torch.Generator().manual_seed(3)).cuda()
    idx = torch.stack([t, live[:70], live[70:140]], 1)
    z = x.detach().double() @ w.detach().double().t() + b.double()
    for tau in (1e-6, 1e-3, 1e3, 1e6):
        loss = linear_distill(x, w, idx, logits, b, temperature=tau, reduction="none")
        lp = torch.log_softmax(logits.double() / tau, 1)
        want = tau * tau * (lp.exp() * (torch.where(lp > -1e300, lp, 0.0) - torch.log_softmax(z / tau, 1).gather(1, idx))).sum(1)
        # logits of magnitudes below 30 (15 of them at most twice over): (D / 16 + 12) 2 u of them twice, times tau; sums and p
        # 300 u of log 300, times tau^2; an exponent's rounding in p, |t| u / tau of an entry whose log q is |z| / tau
        bound = U * (tau * 30 * 30 * 2 + 16 * 30 + tau * tau * 300 * 6)
        assert ((loss.double() - want).abs() <= bound + 4 * U * want.abs()).all(), tau
        dx, = torch.autograd.grad(loss, x, torch.ones_like(loss))
        assert torch.isfinite(dx).all()
    for tau in (0.9e-6, 1.1e6, 1e-300, 1e29):
        with pytest.raises(RuntimeError, match="temperature"):
            linear_distill(x, w, idx, logits, b, temperature=tau)
