"""8-bit activation checkpoints (delrec.checkpoint8) bit for bit against their definition, and
their use in Linear's backward pass and in the model zoo."""

import pytest
import torch

from oracle import sequence_oracle as O

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1,), (33,), (1, 1), (5, 31), (3, 32), (4, 7, 64), (2, 3, 100), (9, 700),
                                   (70001, 3), (2, 40003)])
def test_round_trip(shape, dtype):
    from delrec.checkpoint8 import pack8, unpack8
    g = torch.Generator().manual_seed(shape[-1])
    x = (torch.randn(shape, generator=g) * torch.exp(3 * torch.randn(*shape[:-1], 1, generator=g))).to(dtype)
    p = pack8(x.cuda())
    assert p.q.shape == x.shape and p.e.shape == (*shape[:-1], -(-shape[-1] // 32))
    want = O.restore8(x.double())
    assert torch.equal(unpack8(p, F32).double().cpu(), want)
    assert torch.equal(unpack8(p).cpu(), want.to(dtype))
    assert p.nbytes == p.q.numel() + p.e.numel()


def test_borders():
    """The scale moves where the largest magnitude passes 126 steps; ties go to even; subnormals,
    zeros, the largest values, infinities and NaN."""
    from delrec.checkpoint8 import pack8, unpack8
    rows = []
    for top in (126.0, 126.00001, 125.99999, 127.0, 64.0, 63.999996, 128.0, 1.0, 2.0 ** -120, 2.0 ** -126, 2.0 ** -130,
                2.0 ** -149, 3.0e38, 3.4028234e38, 0.0):
        r = torch.linspace(-1, 1, 32, dtype=torch.float64) * top
        r[3], r[4] = top, -top
        rows.append(r.float())
    half = torch.arange(32).float() + 0.5
    half[0] = 100.0
    rows.append(half)
    x = torch.stack(rows)
    odd = x.clone()
    odd[:, 5], odd[:, 6], odd[:, 7] = float("inf"), float("-inf"), float("nan")
    for v in (x, odd, torch.full((2, 40), float("nan")), torch.full((2, 40), float("inf"))):
        got = unpack8(pack8(v.cuda())).double().cpu()
        assert _same(got, O.restore8(v.double()))
    h = torch.tensor([[65504.0, -65504.0, 6e-8, 1.0]], dtype=F16)
    assert _same(unpack8(pack8(h.cuda()), F32).double().cpu(), O.restore8(h.double()))
    assert _same(unpack8(pack8(h.cuda())).cpu()[:, :2], h[:, :2])     # 64 * 2^10 is past fp16: its largest value
    b = torch.tensor([[3.38e38, -3.38e38, 1e-40, 0.0]], dtype=BF16)
    assert _same(unpack8(pack8(b.cuda()), F32).double().cpu(), O.restore8(b.double()))


def test_spikes_come_back_exactly():
    from delrec.checkpoint8 import pack8, unpack8
    x = (torch.rand(50, 7, 77, device="cuda") < 0.1).float()
    assert torch.equal(unpack8(pack8(x)), x)


def test_layouts_and_empty():
    from delrec.checkpoint8 import Packed8, pack8, unpack8
    x = torch.randn(6, 50, 45, device="cuda")
    a = unpack8(pack8(x.transpose(0, 1)))
    assert torch.equal(a, unpack8(pack8(x.transpose(0, 1).contiguous())))
    off = x.flatten()[3:3 + 64 * 33].view(64, 33)
    assert torch.equal(unpack8(pack8(off)), unpack8(pack8(off.clone())))
    p = pack8(x)
    t = Packed8(p.q.transpose(0, 1), p.e.transpose(0, 1), p.dtype)
    assert torch.equal(unpack8(t), unpack8(p).transpose(0, 1))
    for shape in ((0,), (0, 5), (5, 0)):
        assert unpack8(pack8(torch.empty(shape, device="cuda"))).shape == shape


def _close(a, ref, what):
    scale = ref.abs().max().item() + 1e-30
    err = (a.double().cpu() - ref).abs().max().item() / scale
    assert err < 1e-5, f"{what}: max error {err:.3g} of max |ref|"   # fp32 accuracy, as the projection's own tests


@pytest.mark.parametrize("M,K,N,bias", [(300, 700, 512, True), (777, 1, 10, False), (1500, 130, 70, True),
                                        (64, 31, 8, True), (1, 5, 3, True), (2048, 33, 128, False)])
def test_linear_backward(M, K, N, bias):
    from delrec.linear import linear
    g = torch.Generator().manual_seed(M + K + N)
    x, W = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g) * 0.1
    b = torch.randn(N, generator=g) if bias else None
    gout = torch.randn(M, N, generator=g)
    xd, Wd = x.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
    bd = b.cuda().requires_grad_(True) if bias else None
    out = linear(xd, Wd, bd, binary_input=False, checkpoint8=True)
    _close(out, x.double() @ W.double().t() + (b.double() if bias else 0.0), "out")
    grads = torch.autograd.grad(out, [t for t in (xd, Wd, bd) if t is not None], gout.cuda())
    _close(grads[0], gout.double() @ W.double(), "dx")
    _close(grads[1], gout.double().t() @ O.restore8(x.double()), "dW")
    if bias:
        _close(grads[2], gout.double().sum(0), "db")


def test_linear_spikes_lose_nothing():
    """A spike input gives the bits of the uncompressed forward pass, its gradients to fp32 accuracy, and
    takes a quarter of the bytes."""
    from delrec.linear import Linear
    x = (torch.rand(40, 8, 100, device="cuda") < 0.1).float()
    g = torch.randn(40, 8, 60, device="cuda")
    torch.manual_seed(0)
    lin = Linear(100, 60, binary_input=True).cuda()
    res = []
    for keep in (False, True):
        lin.checkpoint8 = keep
        out = lin(x)
        saved = sum(t.numel() * t.element_size() for t in out.grad_fn.saved_tensors
                    if t is not None and t.shape != lin.weight.shape)
        res.append((saved, out.detach(), *torch.autograd.grad(out, list(lin.parameters()), g)))
    assert torch.equal(res[0][1], res[1][1])
    g2, x2 = g.double().flatten(0, 1).cpu(), x.double().flatten(0, 1).cpu()
    for _, _, dw, db in res:
        _close(dw, g2.t() @ x2, "dW")
        _close(db, g2.sum(0), "db")
    assert res[1][0] <= 0.27 * res[0][0]


@pytest.mark.parametrize("M,K,N", [(5000, 40, 24), (70001, 9, 8)])
def test_linear_weight_gradient_over_many_rows(M, K, N):
    """Sums over many rows: the splits keep the error near that of one."""
    from delrec.linear import linear
    g = torch.Generator().manual_seed(M)
    x, gout = torch.randn(M, K, generator=g), torch.randn(M, N, generator=g)
    W = torch.randn(N, K, generator=g)
    Wd = W.cuda().requires_grad_(True)
    out = linear(x.cuda(), Wd, binary_input=False, checkpoint8=True)
    (dW,) = torch.autograd.grad(out, Wd, gout.cuda())
    _close(dW, gout.double().t() @ O.restore8(x.double()), "dW")


@pytest.mark.parametrize("K", [1, 7, 8, 31, 32, 33, 100, 700])
def test_linear_keeps_what_pack8_keeps(K):
    """The projection's fused 8-bit form is pack8's, infinities and NaN included."""
    from delrec.checkpoint8 import pack8
    from delrec.linear import linear
    x = torch.randn(37, K, device="cuda") * torch.exp(4 * torch.randn(37, 1, device="cuda"))
    x[3, 0], x[5, -1], x[7, K // 2], x[9] = float("inf"), float("-inf"), float("nan"), 0.0
    x[11, 0] = 3.4e38
    W = torch.randn(4, K, device="cuda", requires_grad=True)
    out = linear(x, W, binary_input=False, checkpoint8=True)
    q, _, e = out.grad_fn.saved_tensors
    p = pack8(x)
    assert torch.equal(q, p.q) and torch.equal(e, p.e)


def test_linear_input_gradient_only():
    from delrec.linear import linear
    x = torch.randn(30, 20, device="cuda", requires_grad=True)
    W = torch.randn(10, 20, device="cuda")
    out = linear(x, W, binary_input=False, checkpoint8=True)
    (dx,) = torch.autograd.grad(out, x, torch.ones_like(out))
    _close(dx, (torch.ones(30, 10, dtype=torch.float64) @ W.double().cpu()), "dx")


def test_model_zoo_config():
    """config.checkpoint8 keeps every projection's input in 8 bits; spike inputs: the same output, and
    the gradients to the projections' fp32 accuracy (1e-5) on a path of three of them, twice."""
    from delrec import networks
    from delrec.linear import Linear
    from model_configs import mem_config
    grads = []
    for keep in (False, True):
        cfg = mem_config(hidden=(64, 48), bias=True, T=40, B=16)
        cfg.hybrid_offset_scale = 3
        cfg.checkpoint8 = keep
        torch.manual_seed(0)
        model = networks.SNN_recurrent_hybrid_delays(cfg).cuda()
        assert all(m.checkpoint8 == keep for m in model.layers if isinstance(m, Linear))
        x = (torch.rand(40, 16, cfg.input_size, generator=torch.Generator().manual_seed(5)) < 0.2).float().cuda()
        out = model(x)
        out.sum(0).pow(2).mean().backward()
        grads.append([p.grad for p in model.parameters() if p.grad is not None] + [out.detach()])
    assert len(grads[0]) == len(grads[1]) > 1
    assert torch.equal(grads[0][-1], grads[1][-1])
    for a, b in zip(*grads):
        assert (a - b).abs().max() <= 1e-4 * a.abs().max()
