"""Tokens masked through the bias, by -inf or by the type's lowest value."""

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
