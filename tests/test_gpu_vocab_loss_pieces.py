"""The vocabulary losses past what one pass over the logits' gradient holds, against float64: several pieces of
the vocabulary, more positions than keep a second piece of a 16-bit gradient, tiles of 512 columns, sums in parts."""

import pytest
import torch

from sequence_cases import HALF, within

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

# positions (T, B), D, V, type, entries a teacher keeps (0: cross entropy), temperature, reduction, bias, lengths, least pieces
CASES = [((100, 512), 264, 6007, BF16, 0, 1.0, "mean", True, False, 3), ((100, 512), 40, 6007, F16, 0, 1.0, "none", True, False, 3),
         ((40, 512), 72, 5003, F32, 0, 1.0, "sum", True, False, 3), ((100, 512), 136, 6007, BF16, 7, 2.0, "mean", True, False, 3),
         ((40, 512), 300, 4700, F32, 3, 0.5, "none", True, False, 3), ((64, 1024), 16, 5200, BF16, 0, 1.0, "mean", True, True, 3),
         ((300, 1024), 16, 1100, BF16, 0, 1.0, "sum", True, True, 3),
         ((7, 100), 512, 3001, F16, 20, 1.0, "sum", False, False, 1), ((1, 600), 264, 2049, F32, 64, 2.0, "mean", True, False, 1),
         ((3, 171), 512, 1500, BF16, 33, 1.0, "mean", True, False, 1), ((12, 300), 500, 999, BF16, 5, 1.0, "none", True, True, 1),
         ((1, 513), 24, 260, F16, 4, 1.0, "mean", True, False, 1), ((9, 400), 513, 1111, F16, 1, 3.0, "sum", True, True, 1)]


def _make(case, seed=0):
    (T, B), D, V, dtype, K, tau, reduction, bias, ragged, _ = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    d = dict(x=rnd(T, B, D).to(dtype), w=(rnd(V, D) * 2 * D ** -0.5).to(dtype), bias=rnd(V).to(dtype) if bias else None,
             lengths=torch.randint(0, T + 1, (B,), generator=g, device="cuda") if ragged else None)
    if K:
        d["index"] = torch.randint(0, V, (T, B, K), generator=g, device="cuda")
        d["logits"] = rnd(T, B, K) * 2
        d["index"][torch.rand(T, B, K, generator=g, device="cuda") < 0.1] = -1
    else:
        d["index"] = torch.randint(0, V, (T, B), generator=g, device="cuda")
        d["index"][torch.rand(T, B, generator=g, device="cuda") < 0.1] = -100
    return d, rnd(T, B) if reduction == "none" else torch.tensor(1.7, device="cuda")


def _reference(d, case, grad, split=False):
    """loss, dx, dw, db in float64 and the bounds of fp32 arithmetic with G rounded to its type once (split: and what that
    leaves, once), 4096 positions at a time
    (as ``oracle.selective_oracle.vocab_loss`` has them for small sizes)."""
    (T, B), D, V, dtype, K, tau, reduction, _, _, _ = case
    f, M = torch.float64, T * B
    half = 4 * U if dtype == F32 else HALF[dtype] ** 2 if split else HALF[dtype]
    on = torch.ones(T, B, dtype=torch.bool, device="cuda")
    if d["lengths"] is not None:
        on &= torch.arange(T, device="cuda")[:, None] < d["lengths"][None]
    idx = d["index"].reshape(M, -1)
    on = on.flatten() & (idx >= 0).any(1)
    rows = on.nonzero()[:, 0]
    n = rows.numel()
    w, b = d["w"].to(f), torch.zeros(V, dtype=f, device="cuda") if d["bias"] is None else d["bias"].to(f)
    wa = w.abs()
    share = n if reduction == "mean" else 1
    loss, el = torch.zeros(M, dtype=f, device="cuda"), torch.zeros(M, dtype=f, device="cuda")
    z0 = lambda *s: torch.zeros(*s, dtype=f, device="cuda")   # noqa: E731
    r = dict(dx=z0(M, D), dw=z0(V, D), db=z0(V))
    e = dict(dx=z0(M, D), dw=z0(V, D), db=z0(V))
    c = (grad.reshape(M).to(f) if reduction == "none" else grad.to(f).expand(M) / share) * tau
    top = c[rows].abs().max()
    acc = lambda k: (k / 16 + 24) * 2 * U   # noqa: E731
    for i in range(0, n, 4096):
        at = rows[i:i + 4096]
        x2, ii, cc = d["x"].reshape(M, D)[at].to(f), idx[at], c[at][:, None]
        z = (x2 @ w.t() + b) / tau
        mag = (x2.abs() @ wa.t() + b.abs()) / tau
        ez = (D / 16 + 12) * 2 * U * mag
        et = torch.maximum((D / 32 * 8 + 16) * U * mag, ez)     # a target's logit: a dot product of its own, or the tensor core's
        lse = torch.logsumexp(z, 1)
        elt = 2 * U * (z.abs() + lse.abs()[:, None]) + 100 * U + V / 2048 * U + ez
        q = torch.exp(z - lse[:, None])
        elt = elt + (q * elt).sum(1, keepdim=True)
        kept = ii >= 0
        t = d["logits"].reshape(M, K)[at].to(f) / tau if K else z0(len(at), 1)
        lp = torch.log_softmax(torch.where(kept, t, torch.full_like(t, -float("inf"))), 1)
        p, lp0, ii = torch.exp(lp), torch.where(kept, lp, torch.zeros_like(lp)), ii.clamp(min=0)
        zt = torch.where(kept, z.gather(1, ii), torch.zeros_like(lp))
        rp = (30 + 4 * t.abs().amax(1, keepdim=True) + 2 * lp0.abs()) * U if K else torch.zeros_like(lp)
        loss[at] = tau * tau * ((p * (lp0 - zt)).sum(1) + lse)
        el[at] = tau * tau * ((p * (rp * (1 + lp0.abs() + zt.abs()) + et.gather(1, ii) + (K + 8) * U * (lp0.abs() + zt.abs()))).sum(1)
                              + (q * elt).sum(1) + 8 * U * lse.abs() + 110 * U)
        P = torch.zeros_like(q).scatter_add_(1, ii, p)
        eP = torch.zeros_like(q).scatter_add_(1, ii, p * (rp + (K + 2) * U))
        G = cc * (q - P)
        eG = cc.abs() * (q * (elt + et) + eP + 4 * U * (q + P))
        eG = eG + half * (G.abs() + eG) + top * 2.0 ** -38
        r["dx"][at], e["dx"][at] = G @ w, (eG + acc(V) * G.abs()) @ wa
        r["dw"] += G.t() @ x2
        e["dw"] += (eG + acc(n) * G.abs()).t() @ x2.abs()
        r["db"] += G.sum(0)
        e["db"] += (eG + (n / 128 + 140) * U * G.abs()).sum(0)      # 128 runs of n / 128 rows
    if reduction == "none":
        r["loss"], e["loss"] = loss.view(T, B), el.view(T, B)
    else:
        r["loss"], e["loss"] = loss.sum() / share, el.sum() / share + 4 * U * loss.abs().sum() / share
    r["dx"], e["dx"] = r["dx"].view(T, B, D), e["dx"].view(T, B, D)
    return r, e


def _loss(d, case, **kw):
    from delrec.vocab_loss import linear_cross_entropy, linear_distill
    _, _, _, _, K, tau, reduction, _, _, _ = case
    if K:
        return linear_distill(d["x"], d["w"], d["index"], d["logits"], d["bias"], temperature=tau, reduction=reduction,
                              lengths=d["lengths"], **kw)
    return linear_cross_entropy(d["x"], d["w"], d["index"], d["bias"], reduction=reduction, lengths=d["lengths"], **kw)


@pytest.mark.parametrize("case", CASES)
def test_against_float64(case):
    from delrec import _lib
    pieces = case[-1]
    d, grad = _make(case)
    r, e = _reference(d, case, grad)
    leaves = {k: d[k].requires_grad_(True) for k in ("x", "w", "bias") if d[k] is not None}
    loss = _loss(d, case)
    within(loss, r["loss"], e["loss"], "loss")
    before = _lib.launch_count()
    grads = torch.autograd.grad(loss, list(leaves.values()), grad)
    # a piece takes six or seven launches, all of them three or four more: as many pieces as are meant to be tested
    assert _lib.launch_count() - before > 7 * (pieces - 1) + 4
    for k, v in zip(leaves, grads):
        name = {"x": "dx", "w": "dw", "bias": "db"}[k]
        within(v, r[name], e[name], name)
    for a, v in zip(torch.autograd.grad(_loss(d, case), list(leaves.values()), grad), grads):
        assert torch.equal(a, v)


@pytest.mark.parametrize("case", [c for c in CASES if c[3] != F32])
def test_split_gradient_against_float64(case):
    """Two pieces of a 16-bit gradient: what its rounding adds is squared."""
    d, grad = _make(case, 1)
    r, e = _reference(d, case, grad, True)
    leaves = {k: d[k].requires_grad_(True) for k in ("x", "w", "bias") if d[k] is not None}
    loss = _loss(d, case, split=True)
    assert torch.equal(loss, _loss(d, case))
    for k, v in zip(leaves, torch.autograd.grad(loss, list(leaves.values()), grad)):
        name = {"x": "dx", "w": "dw", "bias": "db"}[k]
        within(v, r[name], e[name], name)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [1, 5, 129, 900])
@pytest.mark.parametrize("K", [1, 2, 8, 9, 31, 32, 33, 128, 129, 1000, 1024])
def test_lists_of_every_length(K, V, dtype):
    """Lists longer and shorter than the vocabulary, most of them with tokens that stand many times."""
    case = ((1, 37), 40, V, dtype, K, 2.0, "none", True, False, 1)
    d, grad = _make(case, 3)
    d["index"][0, 0, 3:] = -1              # a position of three entries at most, one of a single token, one of none
    d["index"][0, 1] = V - 1
    d["index"][0, 2] = -1
    r, e = _reference(d, case, grad)
    leaves = {k: d[k].requires_grad_(True) for k in ("x", "w", "bias")}
    loss = _loss(d, case)
    within(loss, r["loss"], e["loss"], "loss")
    for k, v in zip(leaves, torch.autograd.grad(loss, list(leaves.values()), grad)):
        name = {"x": "dx", "w": "dw", "bias": "db"}[k]
        within(v, r[name], e[name], name)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("positions", [512, 513])
def test_error_of_a_distillation(positions, dtype):
    """Root mean square errors: with two pieces (``split``, or up to 512 positions) that of rounding the result, at most one
    half step evenly (HALF / sqrt(3) of an entry), with one piece as much again at random from the targets' entries."""
    case = ((1, positions), 512, 4000, dtype, 64, 2.0, "mean", False, False, 1)
    d, grad = _make(case, 2)
    r, _ = _reference(d, case, grad)
    leaves = [d[k].requires_grad_(True) for k in ("x", "w")]
    for split in (False, True):
        got = torch.autograd.grad(_loss(d, case, split=split), leaves, grad)
        for v, name in zip(got, ("dx", "dw")):
            ref = r[name]
            err = ((v.double() - ref).pow(2).mean() / ref.pow(2).mean()).sqrt().item()
            one = HALF[dtype] * 3 ** -0.5
            assert err <= (1.02 if split or positions <= 512 else 1.5) * one, (name, split, err / one)
