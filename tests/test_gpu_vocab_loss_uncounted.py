"""Positions that do not count get gradients of 0, whatever gradient the loss itself is given."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("distill", [False, True])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_gradient_without_bounds(reduction, value, distill, dtype):
    from delrec.vocab_loss import linear_cross_entropy, linear_distill
    T, B, D, V = 7, 5, 24, 50
    g = torch.Generator().manual_seed(0)
    x = torch.randn(T, B, D, generator=g).to("cuda", dtype).requires_grad_(True)
    w = torch.randn(V, D, generator=g).to("cuda", dtype).requires_grad_(True)
    b = torch.randn(V, generator=g).to("cuda", dtype).requires_grad_(True)
    lengths = torch.tensor([7, 0, 3, 1, 6], device="cuda")
    t = torch.randint(0, V, (T, B), generator=g).cuda()
    t[2] = -100
    past = (torch.arange(T, device="cuda")[:, None] >= lengths[None]) | (t == -100)

    def call(t):
        if distill:
            return linear_distill(x, w, torch.stack([t, t], -1), torch.zeros(T, B, 2, device="cuda"), b, reduction=reduction,
                                  lengths=lengths)
        return linear_cross_entropy(x, w, t, b, reduction=reduction, lengths=lengths)

    up = torch.tensor(value, device="cuda")
    (dx,) = torch.autograd.grad(call(t), x, up)
    assert (dx[past] == 0).all() and not torch.isfinite(dx[~past]).any()
    # nothing counts: nothing learns
    for v in torch.autograd.grad(call(torch.full_like(t, -100)), (x, w, b), up):
        assert (v == 0).all()
