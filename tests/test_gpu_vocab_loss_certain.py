"""Losses of a vocabulary where the target is all but certain: what is left of the loss and of its gradient
is the difference of two nearly equal numbers, which have to come from one and the same logit."""

import pytest
import torch

from sequence_cases import FLOOR, HALF

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _rows(D, V, dtype, scales, seed=0):
    """x whose row m is along the row of its target in w: logits of scales[m] there and near 0 elsewhere."""
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=g) * D ** -0.5).to(dtype)
    t = torch.randint(0, V, (len(scales),), generator=g)
    x = (w[t].float() * (torch.tensor(scales) / w[t].float().pow(2).sum(1))[:, None]).to(dtype)
    return x, w, t


def _exact(x, w, t):
    """loss and 1 - q of the target in float64, as sums over the other tokens alone, and a bound of the loss."""
    z = x.double() @ w.double().t()
    mag = (x.double().abs() @ w.double().abs().t()).amax(1)
    other = torch.exp(z - z.gather(1, t[:, None]))
    other.scatter_(1, t[:, None], 0.0)
    s = other.sum(1)
    # two logits of the tensor core each off by (D / 16 + 12) 2 u of their products' magnitudes move each share of the
    # sum by that much of itself; the exponents' roundings as much as 4 u |z|.  The sum 1 + s is off by its 1 (an exponential,
    # 4 u), by the sums that the 1 takes part in (10 in each of a tile's four runs of 32 columns, then one to a round of tiles
    # and five) and by the logarithm: 64 u
    rel = 2 * (x.shape[1] / 16 + 12) * 2 * U * mag + 8 * U * z.abs().amax(1) + 100 * U
    loss = torch.log1p(s)
    return loss, s / (1 + s), s * torch.expm1(rel) + 64 * U


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,V", [(512, 4096), (200, 300), (1000, 129)])
def test_loss_of_near_certain_targets(D, V, dtype):
    from delrec.vocab_loss import linear_cross_entropy, linear_distill
    scales = [12.0 + 0.1 * k for k in range(300)]
    x, w, t = _rows(D, V, dtype, scales)
    loss, _, bound = _exact(x, w, t)
    xc, wc, tc = x.cuda(), w.cuda(), t.cuda()
    got = linear_cross_entropy(xc, wc, tc, reduction="none")
    assert (got >= 0).all()
    err = (got.double().cpu() - loss).abs()
    assert (err <= bound + U * loss).all(), f"{(err / bound).max():.3g} of the bound"
    # a teacher that keeps one token is the cross entropy of it, whatever its logit
    one = linear_distill(xc, wc, tc[:, None], torch.randn(300, 1, device="cuda"), reduction="none")
    assert torch.equal(one, got)
    total = linear_cross_entropy(xc, wc, tc, reduction="sum")
    assert abs(total.item() - got.double().sum().item()) <= 2 * U * got.double().sum().item()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tau", [1.0, 2.0])
def test_gradient_of_near_certain_targets(tau, dtype):
    """The target's entry of the logits' gradient, c (q - 1), is what a bias of its token gets from one position: never
    of the wrong sign, however near q is to 1."""
    from delrec.vocab_loss import linear_cross_entropy, linear_distill
    D, V = 512, 2000
    scales = [tau * (9.0 + 2.0 * k) for k in range(16)]
    x, w, t = _rows(D, V, dtype, scales, 1)
    x, w = x.cuda(), w.cuda()
    _, left, bound = _exact((x.double() / tau).cpu(), w.double().cpu(), t)
    for m in range(len(scales)):
        b = torch.zeros(V, dtype=dtype, device="cuda", requires_grad=True)
        if tau == 1.0:
            loss = linear_cross_entropy(x[m:m + 1], w, t[m:m + 1].cuda(), b, reduction="sum")
        else:
            loss = linear_distill(x[m:m + 1], w, t[m:m + 1, None].cuda(), torch.zeros(1, 1, device="cuda"), b, temperature=tau,
                                  reduction="sum")
        (db,) = torch.autograd.grad(loss, b)
        got, want = db[t[m]].item() / tau, -left[m].item()
        assert got <= 0
        # 1 - q = -expm1(-loss) is as far off as the loss; G in two pieces of 16 bits or three, and the result's rounding
        tol = bound[m].item() * 1.01 + (2.0 ** -15 + HALF[dtype]) * abs(want) + torch.finfo(dtype).tiny
        assert abs(got - want) <= tol, (m, got, want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_of_many_near_certain_positions(dtype):
    """More positions than keep a second piece: dx of a position whose loss is nothing is nothing."""
    from delrec.vocab_loss import linear_cross_entropy
    x, w, t = _rows(256, 700, dtype, [20.0 + 0.02 * k for k in range(800)], 2)
    loss, left, bound = _exact(x, w, t)
    xc = x.cuda().requires_grad_(True)
    got = linear_cross_entropy(xc, w.cuda(), t.cuda(), reduction="none")
    (dx,) = torch.autograd.grad(got, xc, torch.ones_like(got))
    z = x.double() @ w.double().t()
    G = torch.softmax(z, 1).scatter_(1, t[:, None], 0.0)
    want = G @ w.double() - left[:, None] * w[t].double()
    # shares of the other tokens good to what the loss is; one rounding each, then the sum's and the result's
    mag = G @ w.double().abs() + left[:, None] * w[t].double().abs()
    rel = (bound / left.clamp(min=1e-30)).clamp(max=1e9)[:, None]
    tol = mag * (rel + HALF[dtype]) * 1.01 + HALF[dtype] * want.abs() + FLOOR[dtype] + 700 * 2.0 ** -38
    assert ((dx.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,K,V", [(2048, 200, 200), (512, 30, 30), (1500, 1000, 1000), (2048, 4, 4)])
def test_distilling_what_the_student_knows(D, K, V, dtype):
    """A teacher that keeps every token, with the student's own logits: the loss is 0, whatever order they come in."""
    from delrec.vocab_loss import linear_distill
    M = 70
    g = torch.Generator().manual_seed(4)
    x, w = torch.randn(M, D, generator=g).to(dtype), (torch.randn(V, D, generator=g) * 8 * D ** -0.5).to(dtype)
    z = x.double() @ w.double().t()
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(M)])
    t = z.gather(1, idx).float()
    got = linear_distill(x.cuda(), w.cuda(), idx.cuda(), t.cuda(), reduction="none").double().cpu()
    # With p = q the errors e_v of the logits move the loss by sum p e - sum q e = 0 and e^2; e is below (D / 16 + 12) 2 u of
    # the products' magnitudes.  What is left: log p is good to (30 + 4 |t| + 2 |log p|) u, the log-sum-exp to
    # (100 + K / 2048) u, log q to 4 u of it, and the products and sums (K / 32 of a lane, then 5) to (K / 32 + 16) u of sum p |log p|.
    lp = torch.log_softmax(z.gather(1, idx), 1)
    p, top = lp.exp(), t.abs().amax(1).double()
    e = (D / 16 + 12) * 2 * U * (x.double().abs() @ w.double().abs().t()).amax(1)
    ent = (p * lp.abs()).sum(1)
    bound = U * (130 + K / 2048 + 4 * top + 6 * ent + (K / 32 + 16) * ent) + 2 * e * e
    assert (got.abs() <= bound).all(), f"{(got / bound).max():.3g} of the bound"
