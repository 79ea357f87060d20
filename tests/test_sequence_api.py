"""The sequence operators' refusals and host-side checks; none needs a GPU."""

import ctypes

import pytest
import torch


def _fake():
    return ctypes.c_void_p(4096)


def test_cpu_tensors_and_bad_types_raise():
    from delrec.block_norm import block_join, block_norm
    from delrec.checkpoint8 import Packed8, pack8, unpack8
    from delrec.gated import gated_scan, gated_step
    from delrec.linear import linear
    t = torch.zeros(3, 2, 4)
    for call in (lambda: gated_scan(t, t), lambda: gated_step(t[0], t[0]), lambda: block_norm(t),
                 lambda: block_join(t, t), lambda: pack8(t), lambda: linear(t, torch.zeros(5, 4)),
                 lambda: unpack8(Packed8(torch.zeros(4, dtype=torch.int8), torch.zeros(1, dtype=torch.uint8),
                                         torch.float32))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="gate_act"):
        block_join(t, t, gate=t, gate_act="relu")
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        unpack8(Packed8(torch.zeros(4, dtype=torch.int8), torch.zeros(1, dtype=torch.uint8), torch.float64))


class _Fake:
    """Stands for a CUDA tensor in the checks that come before any launch."""

    def __init__(self, *shape, dtype=torch.float32, device="cuda:0"):
        self.shape, self.dtype, self.device, self.is_cuda = torch.Size(shape), dtype, device, True

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True


def test_shape_checks():
    from delrec import block_norm, gated
    z = _Fake(5, 2, 12)
    for f in (_Fake(5, 2, 5), _Fake(5, 2, 0), _Fake(4, 2, 12), _Fake(5, 2), _Fake(5, 2, 12, dtype=torch.bfloat16),
              _Fake(5, 2, 24), _Fake(5, 2, 12, device="cuda:1")):
        with pytest.raises(RuntimeError):
            gated.gated_scan(z, f)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        gated.gated_scan(_Fake(5, 2, 12, dtype=torch.float64), _Fake(5, 2, 12, dtype=torch.float64))
    for kw in (dict(h0=_Fake(2, 11)), dict(h0=_Fake(2, 12, dtype=torch.float16)), dict(lengths=_Fake(3)),
               dict(lengths=_Fake(2)), dict(lengths=_Fake(2, dtype=torch.int32, device="cpu")),
               dict(resets=_Fake(5, 2, dtype=torch.uint8)), dict(resets=_Fake(2, 5, dtype=torch.bool))):
        with pytest.raises(RuntimeError):
            gated.gated_scan(z, _Fake(5, 2, 12), **kw)
    s = _Fake(2, 12)
    for kw in (dict(state=_Fake(2, 13)), dict(out=_Fake(3, 12)), dict(active=_Fake(2)),
               dict(active=_Fake(3, dtype=torch.bool))):
        with pytest.raises(RuntimeError):
            gated.gated_step(s, s, **kw)
    x = _Fake(5, 2, 12)
    for args, kw in (((x, _Fake(5, 2, 13)), {}), ((x, x), dict(gate=_Fake(5, 1, 12))), ((x, x, _Fake(11)), {}),
                     ((x, x), dict(scale=_Fake(1))), ((x, x), dict(next_weight=_Fake(12, dtype=torch.bfloat16))),
                     ((x, x), dict(eps=0.0)), ((x, x), dict(eps=float("nan"))), ((x, x), dict(lengths=_Fake(5))),
                     ((x, None), {}), ((x, x), dict(next_weight=_Fake(12), next_norm=False)),
                     ((_Fake(5, 12), _Fake(5, 12)), {})):
        with pytest.raises(RuntimeError):
            block_norm.block_join(*args, **kw)


def test_sizes_past_32_bits_are_refused():
    from delrec import block_norm, checkpoint8, gated
    big = 1 << 31
    for shape in ((big, 1, 4), (1, big, 4), (1, 1, big)):
        t = _Fake(*shape)
        with pytest.raises(RuntimeError, match="32-bit"):
            gated.gated_scan(t, t)
        with pytest.raises(RuntimeError, match="32-bit"):
            block_norm.block_norm(t)
    with pytest.raises(RuntimeError, match="32-bit"):
        checkpoint8.pack8(_Fake(big))


def _scan(**kw):
    from delrec import _lib
    d = dict(T=4, B=2, N=8, G=8, dtype=0)
    d.update(kw)
    return _lib.Scan(d["T"], d["B"], d["N"], d["G"], d["dtype"])


def test_c_entry_points_reject_bad_arguments():
    from delrec import _lib
    lib = _lib.lib()
    p = _fake()

    def fwd(s, z=p, f=p, h=p, q=(None,) * 5):
        return lib.delrec_gated_scan_forward(s and ctypes.byref(s), z, f, None, None, None, h, None, None, *q, None)

    assert fwd(None) == 1
    for bad in (dict(T=0), dict(B=0), dict(N=0), dict(G=0), dict(G=3), dict(dtype=3), dict(dtype=-1), dict(T=-4)):
        assert fwd(_scan(**bad)) == 1
    assert fwd(_scan(), z=None) == 1 and fwd(_scan(), f=None) == 1 and fwd(_scan(), h=None) == 1
    assert fwd(_scan(), q=(p, None, p, p, p)) == 1                 # half of a packed pair
    assert fwd(_scan(G=4), q=(p, p, p, p, p)) == 1                 # packing here is for a gate per channel
    assert fwd(_scan(T=(1 << 30) + 1)) == 4
    assert fwd(_scan(B=1 << 27, N=1024, G=1024)) == 4           # more rows than a grid holds

    def bwd(s, z=p, f=p, qz=None, ez=None, qf=None, ef=None, odd=None, states=p, ws=p, n=1 << 20):
        return lib.delrec_gated_scan_backward(ctypes.byref(s), z, f, qz, ez, qf, ef, odd, None, None, states, p, None,
                                              p, p, None, ws, n, None)

    assert bwd(_scan(), states=None) == 1 and bwd(_scan(), z=None) == 1 and bwd(_scan(), qz=p) == 1
    assert bwd(_scan(), qf=p, ef=p) == 1 and bwd(_scan(G=4), qz=p, ez=p, qf=p, ef=p, odd=p) == 1
    strided = _scan()
    strided.z_t = 1 << 31
    assert fwd(strided) == 4 and bwd(strided) == 4
    wide = _scan(N=128, G=2)
    need = lib.delrec_gated_scan_backward_workspace(ctypes.byref(wide))
    assert need == 4 * 2 * 4 * 2 * 4
    assert bwd(wide, ws=None) == 3 and bwd(wide, n=need - 1) == 3 and bwd(wide, ws=ctypes.c_void_p(4097)) == 3
    assert lib.delrec_gated_scan_backward_workspace(ctypes.byref(_scan())) == 0
    assert lib.delrec_gated_scan_backward_workspace(None) == 0
    step = lambda s, nxt=p: lib.delrec_gated_step(ctypes.byref(s), p, p, None, None, p, nxt, None)   # noqa: E731
    assert step(_scan(T=2)) == 1 and step(_scan(T=1), None) == 1

    def block(**kw):
        d = dict(T=4, B=2, N=8, dtype=0, gate=0, eps=1e-5)
        d.update(kw)
        return _lib.Block(d["T"], d["B"], d["N"], d["dtype"], d["gate"], 0, d["eps"], 0)

    def nf(b, x=p, y=p, u=None, out=p, n=None):
        return lib.delrec_block_norm_forward(ctypes.byref(b), x, y, u, None, None, None, None, out, n, None, None, None)

    for bad in (dict(T=0), dict(N=0), dict(dtype=5), dict(gate=3), dict(gate=-1), dict(eps=0.0), dict(eps=-1.0),
                dict(eps=float("nan"))):
        assert nf(block(**bad)) == 1
    assert nf(block(N=16385)) == 4
    assert nf(block(), x=None) == 1 and nf(block(), out=None) == 1 and nf(block(gate=1)) == 1
    assert nf(block(), y=None, out=None) == 1

    def nb(b, ry=p, rx=p, gn=None, dw=p, ws=p, n=1 << 30, x=p):
        return lib.delrec_block_norm_backward(ctypes.byref(b), x, p, None, None, None, None, None, ry, rx, p, gn, p, p,
                                              None, dw, None, None, ws, n, None)

    assert nb(block(), ry=None) == 1 and nb(block(), rx=None, gn=p) == 1 and nb(block(), x=None, gn=p) == 1
    assert nb(block(), ws=None) == 3 and nb(block(), n=1) == 3
    assert lib.delrec_block_norm_backward_workspace(ctypes.byref(block(N=0))) == 0
    assert lib.delrec_pack8(-1, 4, 0, p, p, p, None) == 1 and lib.delrec_pack8(4, 0, 0, p, p, p, None) == 1
    assert lib.delrec_pack8(4, 4, 7, p, p, p, None) == 1 and lib.delrec_pack8(4, 4, 0, None, p, p, None) == 1
    assert lib.delrec_unpack8(4, 4, 7, p, p, p, None) == 1 and lib.delrec_unpack8(4, 4, 0, p, None, p, None) == 1
    assert lib.delrec_pack8(1 << 61, 4, 0, p, p, p, None) == 1
    assert lib.delrec_linear_backward8(4, 4, 4, None, None, p, p, p, p, None, p, 1 << 20, None) == 1
    assert lib.delrec_linear_backward8(4, 4, 4, p, p, p, p, p, p, None, p, 16, None) == 3
    assert lib.delrec_linear_forward8(4, 4, 4, p, p, None, 0, p, None, p, p, 1 << 20, None) == 1
    assert lib.delrec_linear_forward8(4, 4, 4, p, p, None, 0, p, p, p, p, 16, None) == 3
    assert lib.delrec_linear_backward8_workspace(0, 4, 4) == 0


def test_oracle_restores_within_half_a_step():
    from oracle import sequence_oracle as O
    x = torch.randn(40, 70, dtype=torch.float64) * torch.exp(torch.randn(40, 1, dtype=torch.float64))
    r = O.restore8(x)
    for lo in range(0, 70, 32):
        g, q = x[:, lo:lo + 32], r[:, lo:lo + 32]
        top = g.abs().amax(-1, keepdim=True)
        assert ((g - q).abs() <= top * 2.0 ** -6.9).all()          # half of a step of at most top / 63
    assert torch.equal(O.restore8(r), r)


def test_module_layouts():
    """The modules' parameters and buffers."""
    from delrec.neuron import BlockJoin, BlockNorm, GatedIntegrator
    assert sorted(BlockNorm(8).state_dict()) == ["weight"]
    assert sorted(BlockJoin(8).state_dict()) == ["next_weight", "scale", "weight"]
    assert sorted(BlockJoin(8, next_norm=False).state_dict()) == ["scale", "weight"]
    m = GatedIntegrator()
    assert not m.state_dict() and m.v is None
    with pytest.raises(ValueError):
        GatedIntegrator(step_mode="x")
