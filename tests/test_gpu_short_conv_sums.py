"""Gradients of the convolution's filters over many sequences."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,N", [(4096, 8), (3001, 37)])
def test_filter_gradients_are_rounded_once_over_sequences(B, N):
    """Eight rows of a sequence add up to 8 + k 2^-20 exactly in 24 bits; the sequences' sums, past 24 bits, are added in
    64, so that the gradient is the exact sum rounded."""
    from delrec.short_conv import short_conv
    g = torch.Generator().manual_seed(0)
    x = torch.ones(8, B, N)
    x[0] += torch.randint(0, 1 << 19, (B, N), generator=g).float() * 2.0 ** -20
    w = torch.randn(N, 1, generator=g)
    b = torch.zeros(N)
    xc, wc, bc = x.cuda(), w.cuda().requires_grad_(True), b.cuda().requires_grad_(True)
    y, _ = short_conv(xc, wc, bc, act="none")
    dw, db = torch.autograd.grad(y, (wc, bc), torch.ones_like(y))
    assert torch.equal(dw[:, 0].cpu(), x.double().sum((0, 1)).float())
    assert torch.equal(db.cpu(), torch.full((N,), 8.0 * B))
    y, _ = short_conv(xc, wc, bc, act="none")
    assert torch.equal(torch.autograd.grad(y, bc, xc)[0].cpu(), x.double().sum((0, 1)).float())
