"""Gated linear recurrence over time-major sequences: a leaky integrator whose decay is
learned and input-dependent.

    a = sigmoid(f),   h_t = a_t h_{t-1} + (1 - a_t) z_t      (decay_input=True)
                      h_t = a_t h_{t-1} + z_t                 (decay_input=False)

``decay_input`` has the meaning it has in ``neuron.LIFNode``, whose charge is the case
a = 1 - 1/tau.  ``gated_scan`` runs whole sequences and is differentiable, ``gated_step``
one time step for streaming; both run the library's scan kernels on CUDA tensors of type
float32, bfloat16 or float16, with the state in float32.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib
from .checkpoint8 import Packed8, empty8, pack8, unpack8

SEGMENT = 16     # distance of the states kept for the backward pass


def _check(z, f, dims, layout):
    code = _lib.require_sequence(z)
    zs, fs = z.shape, f.shape
    if len(zs) != dims or len(fs) != dims or zs[:-1] != fs[:-1]:
        raise RuntimeError(f"delrec_b200: z and f must be {layout}, got {tuple(zs)} and {tuple(fs)}")
    if f.dtype != z.dtype or f.device != z.device:
        raise RuntimeError("delrec_b200: z and f must share dtype and device")
    _lib.require_sizes(*zs)
    N, G = zs[-1], fs[-1]
    if N != G and (G == 0 or N % G):
        raise RuntimeError(f"delrec_b200: the {G} gates of f must divide the {N} channels of z")
    return code


def _state(s, B, N, device, name):
    _lib.require_cuda(s)
    if s.shape != (B, N) or s.device != device:
        raise RuntimeError(f"delrec_b200: {name} must be ({B}, {N}) float32 on {device}")


def _forward(z, f, h0, lengths, resets, decay_input, train, keep8):
    """(h, hT, states, 8-bit z and f with their marks or None): one launch."""
    T, B, N = z.shape
    G = f.shape[-1]
    dev = z.device
    h = _lib.empty_rows(z)
    hT = torch.empty(B, N, device=dev)
    states = torch.empty(-(-T // SEGMENT), B, N, device=dev) if train else None
    bits = (None,) * 5
    if keep8 and G == N:
        pz, pf = empty8(z.shape, z.dtype, dev), empty8(f.shape, f.dtype, dev)
        odd = torch.empty(states.shape[0], B, pz.e.shape[-1], dtype=torch.uint8, device=dev)
        bits = (pz.q, pz.e, pf.q, pf.e, odd)
    if T and B and N:
        zt, zb, _ = z.stride()
        ft, fb, _ = f.stride()
        ht, hb, _ = h.stride()
        s = _lib.Scan(T, B, N, G, _lib.SEQ_DTYPES[z.dtype], 1 if decay_input else 0,
                      1 if lengths is not None and lengths.dtype == torch.int64 else 0, 0, zt, zb, ft, fb, ht, hb)
        A = _lib.addr
        _lib.launch("delrec_gated_scan_forward", dev, ctypes.byref(s), z.data_ptr(), f.data_ptr(), A(h0), A(lengths),
                    A(resets), h.data_ptr(), hT.data_ptr(), A(states), A(bits[0]), A(bits[1]), A(bits[2]),
                    A(bits[3]), A(bits[4]))
    elif h0 is not None:
        hT.copy_(h0)
    else:
        hT.zero_()
    return h, hT, states, bits


class GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, f, h0, lengths, resets, decay_input, checkpoint8):
        ctx.set_materialize_grads(False)
        z, f = _lib.rows(z), _lib.rows(f)
        h, hT, states, bits = _forward(z, f, h0, lengths, resets, decay_input, True, checkpoint8)
        ctx.meta = z.shape, f.shape[-1], z.dtype, bool(decay_input), bool(checkpoint8), h0 is not None
        if checkpoint8:
            if bits[0] is None:   # a shared gate is small against its channels: packed apart
                (qz, ez, _), (qf, ef, _) = pack8(z), pack8(f)
                bits = (qz, ez, qf, ef, None)
            ctx.save_for_backward(None, None, states, lengths, resets, *bits)
        else:
            ctx.save_for_backward(z, f, states, lengths, resets, *bits)
        return h, hT

    @staticmethod
    def backward(ctx, *grads):
        # the decorator's bookkeeping is wanted only where a second derivative could be
        return (_once if torch.is_grad_enabled() else _backward)(ctx, *grads)


def _backward(ctx, gh, ghT):
    if gh is None and ghT is None:
        return (None,) * 7
    z, f, states, lengths, resets, qz, ez, qf, ef, odd = ctx.saved_tensors
    (T, B, N), G, dtype, decay_input, keep8, has_h0 = ctx.meta
    if keep8 and odd is None:       # the 8-bit kernel is for a gate per channel
        z, f = unpack8(Packed8(qz, ez, dtype)), unpack8(Packed8(qf, ef, dtype))
        qz = ez = qf = ef = None
    need_z, need_f, need_h = ctx.needs_input_grad[:3]
    like_z, like_f = (qz, qf) if z is None else (z, f)
    dev = states.device
    dz = _lib.empty_rows(like_z, dtype) if need_z else None
    df = _lib.empty_rows(like_f, dtype) if need_f else None
    dh0 = torch.empty(B, N, device=dev) if need_h and has_h0 else None
    if T and B and N:
        if gh is not None:
            gh = _lib.rows(gh)
        if ghT is not None:
            ghT = ghT.contiguous()
        st = []
        for t in (z, f, None, gh, dz, df):
            st += t.stride()[:2] if t is not None else (0, 0)
        s = _lib.Scan(T, B, N, G, _lib.SEQ_DTYPES[dtype], 1 if decay_input else 0,
                      1 if lengths is not None and lengths.dtype == torch.int64 else 0, 0, *st)
        ws, nbytes = None, 0
        if need_f and G != N:
            nbytes = _lib.lib().delrec_gated_scan_backward_workspace(ctypes.byref(s))
            ws = _lib.scratch(nbytes, dev)
        A = _lib.addr
        _lib.launch("delrec_gated_scan_backward", dev, ctypes.byref(s), A(z), A(f), A(qz), A(ez), A(qf), A(ef),
                    A(odd), A(lengths), A(resets), states.data_ptr(), A(gh), A(ghT), A(dz), A(df), A(dh0), A(ws),
                    nbytes)
    else:
        if dh0 is not None:
            dh0 = ghT.clone() if ghT is not None else dh0.zero_()
        if df is not None:
            df.zero_()               # gates without channels: their sums are empty
    return dz, df, dh0, None, None, None, None


_once = once_differentiable(_backward)


def gated_scan(z, f, h0=None, *, lengths=None, resets=None, decay_input=True, checkpoint8=False):
    """Run the recurrence over z (T,B,N) with gate logits f (T,B,G) -> (h (T,B,N), hT (B,N)).

    G divides N: gate g serves the N / G channels from g N / G on (G = N: a gate per
    channel).  ``h0`` (B,N) float32 is the state before the first step (None: 0), ``hT`` the
    float32 state after the last.  ``lengths`` (B,) int32 / int64: sequence b has lengths[b]
    steps; later positions are not read, their h is 0, their gradients are 0, and hT is the
    state after the last step there is.  ``resets`` (T,B) bool: True drops the state before
    that step (sequences packed one after another).  A state that has become infinite stays
    infinite or becomes NaN, up to the next reset.  Strides of T and B are free (a
    batch-major tensor passes as ``.transpose(0, 1)``); a strided channel dimension is copied.

    Gradients reach z, f and h0.  For the backward pass z and f are kept, and the state
    before every 16th step.  ``checkpoint8=True`` keeps z and f in 8 bits instead (see
    ``checkpoint8.pack8``): the forward result is unchanged, the gradients are those of the
    restored z and f, with the states between two kept ones recomputed from them."""
    _check(z, f, 3, "(T, B, N) and (T, B, G)")
    T, B, N = z.shape
    if h0 is not None:
        _state(h0, B, N, z.device, "h0")
    if lengths is not None:
        _lib.require_lengths(lengths, B, z.device)
    if resets is not None:
        if resets.shape != (T, B) or resets.dtype != torch.bool or resets.device != z.device:
            raise RuntimeError(f"delrec_b200: resets must be bool ({T}, {B}) on {z.device}")
        resets = resets.contiguous()
    if torch.is_grad_enabled() and (z.requires_grad or f.requires_grad or (h0 is not None and h0.requires_grad)):
        return GatedScan.apply(z, f, h0, lengths, resets, decay_input, checkpoint8)
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _lib.refuse_tangents(z, f, h0)
    return _forward(_lib.rows(z), _lib.rows(f), h0, lengths, resets, decay_input, False, False)[:2]


def gated_step(z, f, state=None, *, active=None, decay_input=True, out=None):
    """One time step: z (B,N), f (B,G), state (B,N) float32 (None: 0) -> (h (B,N), next state).

    ``out`` receives the next state and may be ``state`` itself (updated in place), but no
    tensor that requires a gradient; None allocates it.  ``active`` (B,) bool: a row with
    False keeps its state and gives h = 0.  No gradient passes; train with ``gated_scan``."""
    code = _check(z, f, 2, "(B, N) and (B, G)")
    B, N = z.shape
    dev = z.device
    if state is not None:
        _state(state, B, N, dev, "state")
    if out is not None:
        _state(out, B, N, dev, "out")
        if torch.is_grad_enabled() and out.requires_grad:
            raise RuntimeError("delrec_b200: out must not require a gradient (no gradient passes)")
    if active is not None:
        if active.shape != (B,) or active.dtype != torch.bool or active.device != dev:
            raise RuntimeError(f"delrec_b200: active must be bool ({B},) on {dev}")
        active = active.contiguous()
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _lib.refuse_tangents(z, f, state)
    z, f = _lib.rows(z), _lib.rows(f)
    h = torch.empty(B, N, device=dev, dtype=z.dtype)
    nxt = torch.empty(B, N, device=dev) if out is None else out
    if B and N:
        s = _lib.Scan(1, B, N, f.shape[1], code, 1 if decay_input else 0, 0, 0, 0, z.stride(0), 0, f.stride(0))
        A = _lib.addr
        _lib.launch("delrec_gated_step", dev, ctypes.byref(s), z.data_ptr(), f.data_ptr(), A(state), A(active),
                    h.data_ptr(), nxt.data_ptr())
    if out is not None:
        increment_version(out)       # who saved the old state for a gradient learns of it
    return h, nxt
