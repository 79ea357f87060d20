"""The refusals and host-side checks of the short convolution, the selective scan and the vocabulary
losses; none needs a GPU."""

import ctypes
import os
import subprocess
import sys

import pytest
import torch


class _Fake:
    """Stands for a CUDA tensor in the checks that come before any launch."""

    def __init__(self, *shape, dtype=torch.float32, device="cuda:0", grad=False):
        self.shape, self.dtype, self.device, self.is_cuda, self.requires_grad = torch.Size(shape), dtype, device, True, grad

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True


def test_import_without_cuda_bindings():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ("import sys, torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda_')]: delattr(torch._C, n)\n"
            "import delrec.short_conv, delrec.selective, delrec.vocab_loss, delrec.neuron\n")
    env = dict(os.environ, PYTHONPATH=os.path.join(root, "snn-delays_b200"))
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr


def test_cpu_tensors_and_bad_types_raise():
    from delrec.selective import selective_scan, selective_step
    from delrec.short_conv import short_conv, short_conv_step
    from delrec.vocab_loss import linear_cross_entropy, linear_distill
    x, w, A, bc = torch.zeros(3, 2, 4), torch.zeros(4, 4), torch.zeros(4, 5), torch.zeros(3, 2, 5)
    t = torch.zeros(3, 2, dtype=torch.int64)
    for call in (lambda: short_conv(x, w), lambda: short_conv_step(x[0], w), lambda: selective_scan(x, x, A, bc, bc),
                 lambda: selective_step(x[0], x[0], A, bc[0], bc[0]), lambda: linear_cross_entropy(x, w, t),
                 lambda: linear_distill(x, w, t.unsqueeze(-1), x[..., :1])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    d = dict(dtype=torch.float64)
    for call in (lambda: short_conv(_Fake(3, 2, 4, **d), _Fake(4, 4)),
                 lambda: selective_scan(_Fake(3, 2, 4, **d), _Fake(3, 2, 4, **d), _Fake(4, 5), bc, bc),
                 lambda: linear_cross_entropy(_Fake(3, 2, 4, **d), _Fake(4, 4, **d), t)):
        with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
            call()


def test_convolution_checks():
    from delrec.short_conv import short_conv, short_conv_step
    x, w = _Fake(5, 2, 12), _Fake(12, 4)
    h = torch.float16
    for args, kw in (((_Fake(5, 12), w), {}), ((x, _Fake(11, 4)), {}), ((x, _Fake(12, 0)), {}), ((x, _Fake(12, 9)), {}),
                     ((x, _Fake(12)), {}), ((x, _Fake(12, 4, dtype=h)), {}), ((x, _Fake(12, 4, device="cuda:1")), {}),
                     ((x, w, _Fake(11)), {}), ((x, w, _Fake(12, dtype=h)), {}), ((x, w, None, _Fake(4, 2, 12)), {}),
                     ((x, w, None, _Fake(3, 2, 12, dtype=h)), {}), ((x, w, None, _Fake(3, 2, 12, device="cuda:1")), {}),
                     ((x, w), dict(act="relu")), ((x, w), dict(lengths=_Fake(3, dtype=torch.int32))),
                     ((x, w), dict(lengths=_Fake(2))), ((x, w), dict(resets=_Fake(2, 5, dtype=torch.bool))),
                     ((x, w), dict(resets=_Fake(5, 2, dtype=torch.uint8)))):
        with pytest.raises(RuntimeError):
            short_conv(*args, **kw)
    s = _Fake(2, 12)
    for args, kw in (((x, w), {}), ((s, w), dict(out=_Fake(4, 2, 12))), ((s, w), dict(out=_Fake(3, 2, 12, dtype=h))),
                     ((s, w), dict(out=_Fake(3, 2, 12, grad=True))), ((s, w), dict(active=_Fake(2))),
                     ((s, w), dict(active=_Fake(3, dtype=torch.bool)))):
        with pytest.raises(RuntimeError):
            short_conv_step(*args, **kw)
    with pytest.raises(RuntimeError, match="32-bit"):
        short_conv(_Fake(1 << 31, 1, 12), w)


def test_selective_checks():
    from delrec.selective import selective_scan, selective_step
    x, A, bc = _Fake(5, 2, 12), _Fake(12, 16), _Fake(5, 2, 16)
    h = torch.float16
    good = (x, x, A, bc, bc)
    bad = [((_Fake(5, 12), x, A, bc, bc), {}), ((x, _Fake(5, 2, 13), A, bc, bc), {}), ((x, _Fake(5, 2, 12, dtype=h), A, bc, bc), {}),
           ((x, x, _Fake(12), bc, bc), {}), ((x, x, _Fake(13, 16), bc, bc), {}), ((x, x, _Fake(12, 0), _Fake(5, 2, 0), _Fake(5, 2, 0)), {}),
           ((x, x, _Fake(12, 129), _Fake(5, 2, 129), _Fake(5, 2, 129)), {}), ((x, x, _Fake(12, 16, dtype=h), bc, bc), {}),
           ((x, x, A, _Fake(5, 2, 15), _Fake(5, 2, 15)), {}), ((x, x, A, bc, _Fake(5, 2, 1, 16)), {}),
           ((x, x, A, _Fake(5, 2, 5, 16), _Fake(5, 2, 5, 16)), {}), ((x, x, A, _Fake(5, 2, 0, 16), _Fake(5, 2, 0, 16)), {}),
           ((x, x, A, _Fake(5, 2, 16, dtype=h), _Fake(5, 2, 16, dtype=h)), {}), ((x, x, A, bc, _Fake(5, 2, 16, device="cuda:1")), {}),
           (good + (_Fake(2, 12, 15),), {}), (good + (_Fake(2, 12, 16, dtype=h),), {}), (good, dict(D=_Fake(11))),
           (good, dict(dt_bias=_Fake(12, dtype=h))), (good, dict(gate=_Fake(5, 2, 11))), (good, dict(gate=_Fake(5, 2, 12, dtype=h))),
           (good, dict(lengths=_Fake(2))), (good, dict(resets=_Fake(5, 3, dtype=torch.bool)))]
    for args, kw in bad:
        with pytest.raises(RuntimeError):
            selective_scan(*args, **kw)
    s, b1 = _Fake(2, 12), _Fake(2, 16)
    for kw in (dict(state=_Fake(2, 12, 15)), dict(out=_Fake(2, 12, 15)), dict(out=_Fake(2, 12, 16, dtype=h)),
               dict(out=_Fake(2, 12, 16, grad=True)), dict(active=_Fake(2)), dict(active=_Fake(3, dtype=torch.bool))):
        with pytest.raises(RuntimeError):
            selective_step(s, s, A, b1, b1, **kw)
    with pytest.raises(RuntimeError):
        selective_step(x, x, A, bc, bc)
    with pytest.raises(RuntimeError, match="32-bit"):
        big = _Fake(1, 1 << 31, 12)
        selective_scan(big, big, A, bc, bc)


def test_loss_checks():
    from delrec.vocab_loss import linear_cross_entropy, linear_distill
    x, w, t = _Fake(5, 2, 12), _Fake(30, 12), _Fake(5, 2, dtype=torch.int64)
    h = torch.float16
    for args, kw in (((_Fake(12), w, _Fake(dtype=torch.int64)), {}), ((x, _Fake(30, 13), t), {}), ((x, _Fake(30, 12, dtype=h), t), {}),
                     ((x, _Fake(0, 12), t), {}), ((x, _Fake(30), t), {}), ((x, _Fake(30, 12, device="cuda:1"), t), {}),
                     ((x, w, _Fake(5, 3, dtype=torch.int64)), {}), ((x, w, _Fake(5, 2)), {}),
                     ((x, w, _Fake(5, 2, dtype=torch.int64, device="cpu")), {}), ((x, w, t, _Fake(29)), {}),
                     ((x, w, t, _Fake(30, dtype=h)), {}), ((x, w, t), dict(reduction="max")), ((x, w, t), dict(ignore_index=1 << 64)),
                     ((x, w, t), dict(lengths=_Fake(5, dtype=torch.int32))), ((x, w, t), dict(lengths=_Fake(2))),
                     ((_Fake(10, 12), w, _Fake(10, dtype=torch.int64)), dict(lengths=_Fake(1, dtype=torch.int32))),
                     ((_Fake(5, 2, 8193), _Fake(30, 8193), t), {}), ((_Fake(1 << 25, 12), w, _Fake(1 << 25, dtype=torch.int64)), {})):
        with pytest.raises(RuntimeError):
            linear_cross_entropy(*args, **kw)
    i, l = _Fake(5, 2, 4, dtype=torch.int32), _Fake(5, 2, 4)
    for args, kw in (((x, w, t, l), {}), ((x, w, _Fake(5, 2, 4), l), {}), ((x, w, _Fake(5, 2, 0, dtype=torch.int32), _Fake(5, 2, 0)), {}),
                     ((x, w, _Fake(5, 2, 1025, dtype=torch.int32), _Fake(5, 2, 1025)), {}), ((x, w, i, _Fake(5, 2, 3)), {}),
                     ((x, w, i, _Fake(5, 2, 4, dtype=torch.float64)), {}), ((x, w, i, l), dict(temperature=0.0)),
                     ((x, w, i, l), dict(temperature=-1.0)), ((x, w, i, l), dict(temperature=float("nan"))),
                     ((x, w, i, l), dict(temperature=float("inf"))), ((x, w, i, l), dict(reduction="max")),
                     ((x, w, i, _Fake(5, 2, 4, grad=True)), {})):
        with pytest.raises(RuntimeError):
            linear_distill(*args, **kw)


def test_c_entry_points_reject_bad_arguments():
    from delrec import _lib
    lib, p = _lib.lib(), ctypes.c_void_p(4096)
    ref = ctypes.byref
    conv = lambda T=4, B=2, N=8, K=4, dtype=0, act=1, kind=0: _lib.Conv(T, B, N, K, dtype, act, kind)   # noqa: E731

    def cf(s, x=p, w=p, y=p):
        return lib.delrec_short_conv_forward(s and ref(s), x, w, None, None, None, None, y, None, None)

    for bad in (None, conv(T=0), conv(B=0), conv(N=-1), conv(K=0), conv(K=9), conv(dtype=3), conv(act=2), conv(kind=3)):
        assert cf(bad) == 1
    assert cf(conv(), x=None) == 1 and cf(conv(), w=None) == 1 and cf(conv(), y=None) == 1
    assert cf(conv(T=(1 << 30) + 1)) == 4
    need = lib.delrec_short_conv_backward_workspace(ref(conv()))
    assert need >= 2 * 5 * 8 * 4 and lib.delrec_short_conv_backward_workspace(None) == 0
    cb = lambda ws, n: lib.delrec_short_conv_backward(ref(conv()), p, p, *(None,) * 4, p, None, p, None, p, None, ws, n, None)   # noqa: E731
    assert cb(None, need) == 3 and cb(p, need - 1) == 3 and cb(ctypes.c_void_p(4097), need) == 3

    sel = lambda T=4, B=2, N=8, S=16, G=1, dtype=0: _lib.Selective(T, B, N, S, G, dtype, 1, 0)   # noqa: E731

    def sf(s, ws=None, n=0, hT=p, **kw):
        a = dict(x=p, dt=p, A=p, Bm=p, Cm=p, y=p)
        a.update(kw)
        return lib.delrec_selective_forward(s and ref(s), a["x"], a["dt"], a["A"], a["Bm"], a["Cm"], *(None,) * 6, a["y"], hT,
                                            None, ws, n, None)

    for bad in (None, sel(T=0), sel(B=0), sel(N=0), sel(S=0), sel(G=0), sel(G=3), sel(dtype=-1)):
        assert sf(bad) == 1
    assert sf(sel(S=129)) == 4 and sf(sel(T=(1 << 30) + 1)) == 4 and sf(sel(B=1 << 20, N=1 << 12)) == 4
    for k in ("x", "dt", "A", "Bm", "Cm", "y", "hT"):
        assert sf(sel(), **{k: None}) == 1
    assert sf(sel(), hT=ctypes.c_void_p(4100)) == 1
    long = sel(T=4096)
    need = lib.delrec_selective_forward_workspace(ref(long))
    assert need > 0 and lib.delrec_selective_forward_workspace(ref(sel())) == 0
    assert sf(long) == 3 and sf(long, ws=p, n=need - 1) == 3 and sf(long, ws=ctypes.c_void_p(4097), n=need) == 3
    need = lib.delrec_selective_backward_workspace(ref(sel()))
    sb = lambda states=p, ws=p, n=need, dgate=None: lib.delrec_selective_backward(   # noqa: E731
        ref(sel()), p, p, p, p, p, None, None, None, None, None, states, p, None, p, p, p, p, p, None, dgate, None, None, ws, n, None)
    assert sb(states=None) == 1 and sb(dgate=p) == 1 and sb(ws=None) == 3 and sb(n=need - 1) == 3
    step = lambda s: lib.delrec_selective_step(ref(s), p, p, p, p, p, *(None,) * 5, p, p, None)   # noqa: E731
    assert step(sel(T=2)) == 1 and step(sel(T=1, S=129)) == 4

    def voc(T=4, B=2, D=16, V=100, K=1, dtype=0, distill=0, reduction=1, teacher=0, tau=1.0):
        return _lib.Vocab(T, B, D, V, K, dtype, distill, reduction, 0, 0, teacher, 1, tau, 0, -100, B * D, D)

    def vf(s, keep=p, nk=1 << 40, ws=p, n=1 << 40, logits=None, index=p, w=p):
        return lib.delrec_vocab_loss_forward(s and ref(s), p, w, None, index, logits, None, p, keep, nk, ws, n, None)

    for bad in (None, voc(T=0), voc(B=0), voc(D=0), voc(V=0), voc(K=0), voc(K=2), voc(dtype=4), voc(reduction=3), voc(tau=0.0),
                voc(tau=float("nan")), voc(distill=1, teacher=5)):
        assert vf(bad) == 1
        assert lib.delrec_vocab_loss_keep(bad and ref(bad)) == 0
    assert vf(voc(D=8193)) == 4 and vf(voc(K=1025, distill=1)) == 4 and vf(voc(T=1 << 24)) == 4
    assert vf(voc(), index=None) == 1 and vf(voc(distill=1)) == 1 and vf(voc(), w=ctypes.c_void_p(4100)) == 1
    need, keep = lib.delrec_vocab_loss_forward_workspace(ref(voc())), lib.delrec_vocab_loss_keep(ref(voc()))
    assert vf(voc(), ws=None) == 3 and vf(voc(), n=need - 1) == 3 and vf(voc(), nk=keep - 1) == 3 and vf(voc(), keep=None) == 3
    need = lib.delrec_vocab_loss_backward_workspace(ref(voc()))
    vb = lambda g=p, db=None, n=need, ws=p: lib.delrec_vocab_loss_backward(   # noqa: E731
        ref(voc()), p, p, None, g, p, keep, p, p, db, ws, n, None)
    assert vb(g=None) == 1 and vb(db=p) == 1 and vb(n=need - 1) == 3 and vb(ws=None) == 3


def test_the_logits_gradient_stays_within_its_room():
    """The scratch of a backward pass does not grow with positions times vocabulary."""
    from delrec import _lib
    lib = _lib.lib()
    s = _lib.Vocab(64, 1024, 512, 65536, 1, 1, 0, 1, 0, 0, 0, 1, 1.0, 0, -100, 512, 512)
    whole = 65536 * 65536 * 2
    assert lib.delrec_vocab_loss_backward_workspace(ctypes.byref(s)) < whole / 8
    assert lib.delrec_vocab_loss_forward_workspace(ctypes.byref(s)) < whole / 8


def test_room_of_the_logits_gradient():
    """256 MB of it, or 512 columns of all positions where those take more: what a backward pass takes besides is the same
    for a vocabulary of one such piece and of many, but for the weight's operand and sums."""
    from delrec import _lib
    lib = _lib.lib()

    def take(M, V, dtype):
        s = _lib.Vocab(1, M, 8, V, 1, dtype, 0, 1, 0, 0, 0, 1, 1.0, 0, -100, 0, 8)
        return lib.delrec_vocab_loss_backward_workspace(ctypes.byref(s))

    for dtype, each in ((1, 2), (2, 2), (0, 6)):
        for M in (600, 51200, 100000, 262144, 300000, 1 << 20):
            Mp = (M + 255) // 256 * 256
            room = max(256 << 20, 512 * Mp * each)
            V = 64 * max(512, room // (Mp * each))       # many pieces of it
            if (M // 256 + 1) * (V // 128 + 1) > 1 << 27:
                continue
            # x's operand, dx's and dweight's sums in up to 16 parts, dbias's runs, and the weight's operand
            rest = Mp * 8 * (each + 16 * 4) + V * 8 * each + (room // (Mp * each) + 256) * (16 * 8 * 4 + 128 * 4) + Mp * 4 + 4096
            assert 0 < take(M, V, dtype) <= room + rest, (dtype, M)


def test_room_of_the_scans_sums():
    """dB and dC have a place for their sums to each tile of channels, but no more than one to 16 channels where that fills
    the GPU eight times, and none where neither is wanted."""
    from delrec import _lib
    lib, p = _lib.lib(), ctypes.c_void_p(4096)

    def take(T, B, N, S, G=1, no_bc=0):
        s = _lib.Selective(T, B, N, S, G, 0, 1, 0, 0, no_bc)
        return lib.delrec_selective_backward_workspace(ctypes.byref(s))

    for T, B, N, S, G, places in ((250, 256, 2048, 128, 1, 128), (250, 256, 512, 16, 1, 8), (9, 4000, 64, 100, 1, 4),
                                  (64, 600, 64, 128, 1, 8), (100, 256, 4096, 64, 4, 64)):
        none = take(T, B, N, S, G, 1)
        # dA, dD and dbias to each sequence and chunk (one chunk here)
        assert B * N * (S + 2) * 4 <= none <= B * N * (S + 2) * 4 + 4096
        assert take(T, B, N, S, G) - none <= 2 * places * T * B * G * S * 4 + 1024
    s = _lib.Selective(4, 2, 8, 16, 1, 0, 1, 0, 0, 1)
    need = take(4, 2, 8, 16)
    for dB, dC in ((p, None), (None, p)):
        assert lib.delrec_selective_backward(ctypes.byref(s), p, p, p, p, p, *(None,) * 5, p, p, None, p, p, p, dB, dC, None, None,
                                             None, None, p, need, None) == 1
