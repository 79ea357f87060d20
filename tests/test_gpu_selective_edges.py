"""The selective scan at decays without bounds and with many channels to a sequence."""

import pytest
import torch

from sequence_cases import within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
KEYS = ("x", "dt", "A", "Bm", "Cm", "h0", "D", "gate", "dt_bias")


def _inputs(T, B, N, S, dtype, lengths, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    d = dict(x=rnd(T, B, N).to(dtype), dt=rnd(T, B, N).to(dtype), A=-rnd(N, S).abs() - 0.1, Bm=rnd(T, B, S).to(dtype),
             Cm=rnd(T, B, S).to(dtype), h0=rnd(B, N, S), D=rnd(N), gate=rnd(T, B, N).to(dtype), dt_bias=rnd(N))
    d = {k: v.cuda() for k, v in d.items()}
    return d, torch.tensor(lengths, device="cuda") if lengths else None, rnd(T, B, N).to(dtype).cuda(), rnd(B, N, S).cuda()


def _run(d, lengths, gy, gh, **kw):
    from delrec.selective import selective_scan
    c = {k: v.detach().clone().requires_grad_(True) for k, v in d.items()}
    y, hT = selective_scan(c["x"], c["dt"], c["A"], c["Bm"], c["Cm"], c["h0"], D=c["D"], gate=c["gate"], dt_bias=c["dt_bias"],
                           lengths=lengths, **kw)
    return [y, hT, *torch.autograd.grad((y, hT), [c[k] for k in KEYS], (gy, gh))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,N,S,lengths", [(13, 2, 6, 5, [13, 3]), (8, 1, 4, 16, None), (9, 3, 40, 4, [0, 9, 1]),
                                             (300, 2, 8, 16, [300, 77]), (515, 1, 5, 1, None)])
def test_a_decay_of_minus_infinity_drops_the_state(T, B, N, S, lengths, dtype):
    """A = -inf (what -exp(A_log) gives past A_log = 88.7) is a decay of 0 in every step there is: the bits of A = -1e30,
    whose decay is 0 as well, and no trace in the steps that there are not."""
    d, lengths, gy, gh = _inputs(T, B, N, S, dtype, lengths)
    hit = torch.rand(N, S, generator=torch.Generator().manual_seed(1)).cuda() < 0.4
    hit[0, 0] = True
    big = dict(d, A=torch.where(hit, torch.full_like(d["A"], -1e30), d["A"]))
    inf = dict(d, A=torch.where(hit, torch.full_like(d["A"], -float("inf")), d["A"]))
    for got, want, name in zip(_run(inf, lengths, gy, gh), _run(big, lengths, gy, gh), ("y", "hT") + KEYS):
        assert torch.isfinite(want).all() and torch.equal(got, want), name
    # by the formula: such a state is the last step's input alone, or the first state where there is no step
    hT = _run(inf, lengths, gy, gh)[1].detach().double()
    for b in range(B):
        n = T if lengths is None else int(lengths[b])
        if n == 0:
            assert torch.equal(hT[b], d["h0"][b].double())
            continue
        delta = torch.nn.functional.softplus(d["dt"][n - 1, b].double() + d["dt_bias"].double())
        want = (delta * d["x"][n - 1, b].double())[:, None] * d["Bm"][n - 1, b].double()
        # delta good to (10 + |z|) u, three products
        assert ((hT[b] - want).abs()[hit] <= (32 * 2.0 ** -24 * want.abs())[hit] + 2.0 ** -140).all()


@pytest.mark.parametrize("B", [2, 9000])
def test_a_step_with_a_decay_of_minus_infinity(B):
    """Also where there are more sequences than threads."""
    from delrec.selective import selective_scan, selective_step
    d, _, _, _ = _inputs(1, B, 24, 8, torch.float32, None)
    d["A"][::3, ::2] = -float("inf")
    y, h = selective_step(d["x"][0], d["dt"][0], d["A"], d["Bm"][0], d["Cm"][0], d["h0"], D=d["D"], gate=d["gate"][0],
                          dt_bias=d["dt_bias"])
    ys, hs = selective_scan(d["x"], d["dt"], d["A"], d["Bm"], d["Cm"], d["h0"], D=d["D"], gate=d["gate"], dt_bias=d["dt_bias"])
    assert torch.isfinite(y).all() and torch.equal(h, hs)
    torch.testing.assert_close(y, ys[0], rtol=2.0 ** -18, atol=2.0 ** -18)     # the order of a sum of eight
