"""The gated scan's kernel variants that need many rows or long sequences, against the float64 loop:
blocks of a cluster that share a row's time, two channels to a lane, segments of 32 steps, 8-bit
checkpoints with infinities and at the largest scale.  Bounds as in test_gpu_gated.

What the sizes reach (the launch's rules; S = ceil(T / 16) segments, 8 warps a block): clusters
where ceil(N / 32) rows of tiles leave SMs empty; two channels to a lane for 16-bit rows of 16-byte
multiples with B ceil(N / 64) min(16, ceil(S / 8)) >= 296; segments of 32 steps for others in
clusters of c blocks with S >= 16 c."""

import pytest
import torch

from oracle import sequence_oracle as O
from sequence_cases import within
from test_gpu_gated import _check, _cuda, _inputs

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,N", [(260, 32), (700, 40), (1500, 32), (4200, 32)])
def test_cluster_blocks_past_the_sequence_end(T, N, dtype):
    """Rows much shorter than T: the blocks of a cluster that lie past a row's end reach the exchange
    long before the others have loaded anything.  Launched back to back, the results stay those of the
    first time, which are the oracle's."""
    from delrec.gated import gated_scan
    c = _inputs(T, 6, N, 1, dtype, ragged=True, resets=True)
    c["lengths"][:6] = torch.tensor([0, 1, 17, T, 130, T // 2])
    first = _check(c)
    d = _cuda(c)
    z, f, h0 = (d[k].requires_grad_(True) for k in ("z", "f", "h0"))
    for _ in range(20):
        h, hT = gated_scan(z, f, h0, lengths=d["lengths"].int(), resets=d["resets"])
        grads = torch.autograd.grad((h, hT), (z, f, h0), (d["gh"], d["ghT"]))
        for got, want in zip((h, hT, *grads), (first[0], first[1], *first[2])):
            assert torch.equal(got, want)


@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("with_gh", [True, False])
def test_c_buffers_at_odd_addresses(keep8, with_gh):
    """States 4 bytes and codes one byte past an aligned address: a C caller's buffers promise no more than
    their element's alignment, whatever the sizes lead to (here two channels to a lane)."""
    import ctypes
    from delrec import _lib
    T, B, N = 40, 5, 64 * 60 + 16
    c = _inputs(T, B, N, 1, BF16)
    d = _cuda(c)
    lib, S, G = _lib.lib(), -(-T // 16), -(-N // 32)

    def odd(*shape, dtype=torch.float32):
        return torch.zeros(torch.Size(shape).numel() + 1, dtype=dtype, device="cuda")[1:].view(shape)

    h = torch.empty(T, B, N, dtype=BF16, device="cuda")
    hT, states = odd(B, N), odd(S, B, N)
    q = [odd(T, B, N, dtype=torch.int8), odd(T, B, G, dtype=torch.uint8), odd(T, B, N, dtype=torch.int8),
         odd(T, B, G, dtype=torch.uint8), odd(S, B, G, dtype=torch.uint8)] if keep8 else [None] * 5
    assert states.data_ptr() % 8 == 4 and (not keep8 or q[0].data_ptr() % 2 == 1)
    A, stream = _lib.addr, torch.cuda.current_stream().cuda_stream
    s = _lib.Scan(T, B, N, N, 1, 1, 0, 0, *(B * N, N) * 6)
    assert lib.delrec_gated_scan_forward(ctypes.byref(s), A(d["z"]), A(d["f"]), A(d["h0"]), None, None, A(h), A(hT),
                                         A(states), *map(A, q), stream) == 0
    dz, df, dh0 = torch.empty_like(h), torch.empty_like(h), odd(B, N)
    zf = [None, None] if keep8 else [A(d["z"]), A(d["f"])]
    assert lib.delrec_gated_scan_backward(ctypes.byref(s), *zf, *map(A, q), None, None, A(states),
                                          A(d["gh"]) if with_gh else None, A(d["ghT"]), A(dz), A(df), A(dh0), None, 0,
                                          stream) == 0
    r = O.gated_scan(c["z"], c["f"], c["h0"])
    within(h, r["h"], r["err"], "h")
    within(hT, r["hT"], r["errT"], "hT")
    z, f, pre = c["z"].double(), c["f"].double(), r["pre"]
    perr = torch.zeros_like(pre)
    perr[1:] = r["err"][:-1]
    if keep8:
        z, f = O.restore8(z), O.restore8(f)
        pre, e = O.recompute(z, f, pre)
        perr = e + perr[torch.arange(T) // 16 * 16]
        for got, e8, ref in ((q[0], q[1], z), (q[2], q[3], f)):
            scale = ((e8.long().cpu() + (1023 - 127)) << 52).view(torch.float64).repeat_interleave(32, -1)[..., :N]
            assert torch.equal(got.double().cpu() * scale, ref)
    b = O.gated_scan_backward(z, f, pre, perr, c["gh"] if with_gh else torch.zeros_like(c["gh"]), c["ghT"])
    within(dz, b["dz"], b["ez"], "dz")
    within(df, b["df"], b["ef"], "df")
    within(dh0, b["dh0"], b["e0"], "dh0")


# (T, B, N): rows of two channels to a lane; one block a row, two and four blocks a row
TWO = [(20, 5, 64 * 60 + 8), (150, 5, 64 * 30 + 40), (264, 5, 64 * 20), (600, 4, 64 * 20 - 8)]


@pytest.mark.parametrize("decay_input", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,B,N", TWO)
def test_two_channels_to_a_lane(T, B, N, dtype, decay_input):
    c = _inputs(T, B, N, 1, dtype, ragged=True, resets=True)
    c["lengths"][:4] = torch.tensor([T, 0, 17, T - 1])
    _check(c, decay_input)
    c["lengths"] = c["resets"] = None
    _check(c, decay_input)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,B,N", [(20, 5, 64 * 60 + 16), (150, 5, 64 * 30 + 32), (264, 5, 64 * 20), (150, 5, 64 * 30 + 40)])
def test_two_channels_to_a_lane_checkpoint8(T, B, N, dtype):
    c = _inputs(T, B, N, 1, dtype, ragged=True, resets=True)
    c["lengths"][:4] = torch.tensor([T, 0, 17, T - 1])
    _check(c, checkpoint8=True)
    _check(c, decay_input=False, checkpoint8=True)
    c["lengths"] = c["resets"] = None
    _check(c, checkpoint8=True)


# segments of 32 steps: clusters of 16 blocks, and of two
@pytest.mark.parametrize("decay_input", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,B,N", [(4200, 2, 40), (4111, 1, 32), (500, 4, 1120)])
def test_segments_of_32_steps(T, B, N, dtype, decay_input):
    c = _inputs(T, B, N, 1, dtype, mean=4.0)
    _check(c, decay_input)
    if B > 1:
        c = _inputs(T, B, N, 1, dtype, ragged=True, resets=True, mean=4.0)
        c["lengths"][:2] = torch.tensor([T - 13, 45])
        _check(c, decay_input)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,B,N", [(45, 3, 40), (150, 3, 64), (150, 5, 64 * 30 + 32)])
def test_checkpoint8_with_infinities_and_large_values(T, B, N, dtype):
    """Codes that stand for infinities and NaN (the slow forms of packing and of the walk), and groups at
    the largest scale, whose codes are cut.  The rest of z is as ever; a reset a few steps on keeps what
    is not finite short.  The large values are positive and meet gradients below 2^-6, so that
    a (1 - a) G (h - z) stays in range."""
    c = _inputs(T, B, N, 1, dtype)
    c["resets"] = torch.zeros(T, B, dtype=torch.bool)
    for b, t, n, value in ((0, 3, 5, float("inf")), (1, 18, 33, float("-inf")), (2, 31, 0, float("nan")),
                           (0, T - 9, 32, float("nan"))):
        c["z"][t, b, n] = value
        c["resets"][t + 4, b] = True
    big = slice(32, 36)
    c["z"][20:24, 0, big] = torch.tensor([3.39e38, 3.37e38, 2e38, 1e37]).to(dtype)
    c["h0"][0, big] = c["h0"][0, big].abs()
    c["resets"][24, 0] = True
    c["gh"] *= 2.0 ** -9
    c["ghT"] *= 2.0 ** -9
    from delrec.gated import gated_scan
    d = _cuda(c)
    leaves = [d[k].requires_grad_(True) for k in ("z", "f", "h0")]
    h, hT = gated_scan(*leaves, resets=d["resets"], checkpoint8=True)
    grads = torch.autograd.grad((h, hT), leaves, (d["gh"], d["ghT"]))
    r = O.gated_scan(c["z"], c["f"], c["h0"], resets=c["resets"])
    within(h, r["h"], r["err"], "h")
    within(hT, r["hT"], r["errT"], "hT")
    z, f = O.restore8(c["z"].double()), O.restore8(c["f"].double())
    pre, perr = O.recompute(z, f, r["pre"], resets=c["resets"])
    # A kept state's bound rides along inside its segment, up to the first reset: behind one the state
    # does not depend on it (and a bound of a state that is not finite is none).
    seg = torch.arange(T) // 16 * 16
    cut = torch.stack([c["resets"][int(s):t].any(0) for t, s in enumerate(seg)])        # a reset before step t
    kept = torch.cat([torch.zeros_like(r["err"][:1]), r["err"][:-1]])[seg]
    perr = perr + torch.where(cut[..., None], torch.zeros_like(kept), kept)
    b = O.gated_scan_backward(z, f, pre, perr, c["gh"], c["ghT"], resets=c["resets"])
    for got, k, e in zip(grads, ("dz", "df", "dh0"), ("ez", "ef", "e0")):
        within(got, b[k], b[e], k)
