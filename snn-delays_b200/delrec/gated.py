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
from torch.autograd.function import once_differentiable

from . import _lib
from .checkpoint8 import Packed8, empty8, pack8, unpack8

SEGMENT = 16     # distance of the states kept for the backward pass


def _check(z, f, dims, layout):
    code = _lib.require_sequence(z, f)
    if z.dim() != dims or f.dim() != dims or z.shape[:-1] != f.shape[:-1]:
        raise RuntimeError(f"delrec_b200: z and f must be {layout}, got {tuple(z.shape)} and {tuple(f.shape)}")
    if f.dtype != z.dtype or f.device != z.device:
        raise RuntimeError("delrec_b200: z and f must share dtype and device")
    N, G = z.shape[-1], f.shape[-1]
    if G == 0 or N % G:
        if N or G:
            raise RuntimeError(f"delrec_b200: the {G} gates of f must divide the {N} channels of z")
    return code


def _state(s, B, N, z, name):
    if s is not None:
        _lib.require_cuda(s)
        if s.shape != (B, N) or s.device != z.device:
            raise RuntimeError(f"delrec_b200: {name} must be ({B}, {N}) float32 on {z.device}")


class GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, f, h0, lengths, resets, decay_input, checkpoint8):
        T, B, N = z.shape
        G = f.shape[-1]
        ctx.set_materialize_grads(False)
        z, f = _lib.rows(z.detach()), _lib.rows(f.detach())
        dev = z.device
        h = _lib.empty_rows(z)
        hT = torch.empty(B, N, device=dev)
        train = any(ctx.needs_input_grad[:3])
        s = _lib.Scan(T, B, N, G, _lib.SEQ_DTYPES[z.dtype], int(decay_input),
                      int(lengths is not None and lengths.dtype == torch.int64), 0,
                      *z.stride()[:2], *f.stride()[:2], *h.stride()[:2])
        states = torch.empty(-(-T // SEGMENT), B, N, device=dev) if train else None
        keep8 = bool(checkpoint8) and train
        pz = pf = odd = None
        if keep8 and G == N:
            pz, pf = empty8(z.shape, z.dtype, dev), empty8(f.shape, f.dtype, dev)
            odd = torch.empty(*states.shape[:2], pz.e.shape[-1], dtype=torch.uint8, device=dev)
        if T and B and N:
            with _lib.on_device(z):
                _lib.check(_lib.lib().delrec_gated_scan_forward(
                    ctypes.byref(s), z.data_ptr(), f.data_ptr(), _lib.addr(h0), _lib.addr(lengths),
                    _lib.addr(resets), h.data_ptr(), hT.data_ptr(), _lib.addr(states),
                    _lib.addr(pz and pz.q), _lib.addr(pz and pz.e), _lib.addr(pf and pf.q),
                    _lib.addr(pf and pf.e), _lib.addr(odd), _lib.stream_ptr(dev)), "delrec_gated_scan_forward")
        elif h0 is not None:
            hT.copy_(h0.detach())
        else:
            hT.zero_()
        if not train:
            return h, hT
        if keep8:
            if pz is None:   # a shared gate is small against its channels: packed apart
                pz, pf = pack8(z), pack8(f)
            ctx.save_for_backward(pz.q, pz.e, pf.q, pf.e, odd, states, lengths, resets)
        else:
            ctx.save_for_backward(z, f, states, lengths, resets)
        ctx.scan, ctx.keep8, ctx.dtype = s, keep8, z.dtype
        ctx.has_h0 = h0 is not None
        return h, hT

    @staticmethod
    @once_differentiable
    def backward(ctx, gh, ghT):
        z = f = pz = pf = odd = None
        if ctx.keep8:
            qz, ez, qf, ef, odd, states, lengths, resets = ctx.saved_tensors
            pz, pf = Packed8(qz, ez, ctx.dtype), Packed8(qf, ef, ctx.dtype)
            if ctx.scan.G != ctx.scan.N:    # the 8-bit kernel is for a gate per channel
                z, f, pz, pf = unpack8(pz), unpack8(pf), None, None
            like_z, like_f = qz, qf
        else:
            z, f, states, lengths, resets = ctx.saved_tensors
            like_z, like_f = z, f
        if gh is None and ghT is None:
            return (None,) * 7
        dev = like_z.device
        T, B, N = like_z.shape
        if gh is not None:
            gh = _lib.rows(gh)
        if ghT is not None:
            ghT = ghT.contiguous()
        need_z, need_f, need_h = ctx.needs_input_grad[:3]
        dz = _lib.empty_rows(like_z, ctx.dtype) if need_z else None
        df = _lib.empty_rows(like_f, ctx.dtype) if need_f else None
        dh0 = torch.empty(B, N, device=dev) if need_h and ctx.has_h0 else None
        if T and B and N:
            # a copy of the descriptor: two backward passes of one graph may run at once
            s = _lib.Scan.from_buffer_copy(ctx.scan)
            for name, t in (("z", z), ("f", f), ("gh", gh), ("dz", dz), ("df", df)):
                if t is not None:
                    setattr(s, name + "_t", t.stride(0))
                    setattr(s, name + "_b", t.stride(1))
            lib = _lib.lib()
            nbytes = lib.delrec_gated_scan_backward_workspace(ctypes.byref(s)) if need_f else 0
            ws = _lib.scratch(nbytes, dev)
            with _lib.on_device(like_z):
                _lib.check(lib.delrec_gated_scan_backward(
                    ctypes.byref(s), _lib.addr(z), _lib.addr(f), _lib.addr(pz and pz.q), _lib.addr(pz and pz.e),
                    _lib.addr(pf and pf.q), _lib.addr(pf and pf.e), _lib.addr(odd), _lib.addr(lengths), _lib.addr(resets),
                    states.data_ptr(), _lib.addr(gh), _lib.addr(ghT), _lib.addr(dz), _lib.addr(df),
                    _lib.addr(dh0), _lib.addr(ws), nbytes, _lib.stream_ptr(dev)), "delrec_gated_scan_backward")
        elif dh0 is not None:
            dh0 = ghT.clone() if ghT is not None else dh0.zero_()
        return dz, df, dh0, None, None, None, None


def gated_scan(z, f, h0=None, *, lengths=None, resets=None, decay_input=True, checkpoint8=False):
    """Run the recurrence over z (T,B,N) with gate logits f (T,B,G) -> (h (T,B,N), hT (B,N)).

    G divides N: gate g serves the N / G channels from g N / G on (G = N: a gate per
    channel).  ``h0`` (B,N) float32 is the state before the first step (None: 0), ``hT`` the
    float32 state after the last.  ``lengths`` (B,) int32 / int64: sequence b has lengths[b]
    steps; later positions are not read, their h is 0, their gradients are 0, and hT is the
    state after the last step there is.  ``resets`` (T,B) bool: True drops the state before
    that step (sequences packed one after another).  Strides of T and B are free (a
    batch-major tensor passes as ``.transpose(0, 1)``); a strided channel dimension is copied.

    Gradients reach z, f and h0.  For the backward pass z and f are kept, and the state
    before every 16th step.  ``checkpoint8=True`` keeps z and f in 8 bits instead (see
    ``checkpoint8.pack8``): the forward result is unchanged, the gradients are those of the
    restored z and f, with the states between two kept ones recomputed from them."""
    _check(z, f, 3, "(T, B, N) and (T, B, G)")
    T, B, N = z.shape
    _state(h0, B, N, z, "h0")
    if lengths is not None:
        _lib.require_lengths(lengths, B, z.device)
    if resets is not None:
        if resets.shape != (T, B) or resets.dtype != torch.bool or resets.device != z.device:
            raise RuntimeError(f"delrec_b200: resets must be bool ({T}, {B}) on {z.device}")
        resets = resets.contiguous()
    return GatedScan.apply(z, f, h0, lengths, resets, decay_input, checkpoint8)


def gated_step(z, f, state=None, *, active=None, decay_input=True, out=None):
    """One time step: z (B,N), f (B,G), state (B,N) float32 (None: 0) -> (h (B,N), next state).

    ``out`` receives the next state and may be ``state`` itself (updated in place); None
    allocates it.  ``active`` (B,) bool: a row with False keeps its state and gives h = 0.
    No gradient passes; train with ``gated_scan``."""
    code = _check(z, f, 2, "(B, N) and (B, G)")
    B, N = z.shape
    _state(state, B, N, z, "state")
    _state(out, B, N, z, "out")
    if active is not None:
        if active.shape != (B,) or active.dtype != torch.bool or active.device != z.device:
            raise RuntimeError(f"delrec_b200: active must be bool ({B},) on {z.device}")
        active = active.contiguous()
    z, f = _lib.rows(z.detach()), _lib.rows(f.detach())
    h = torch.empty(B, N, device=z.device, dtype=z.dtype)
    nxt = torch.empty(B, N, device=z.device) if out is None else out
    if B and N:
        s = _lib.Scan(1, B, N, f.shape[1], code, int(decay_input), 0, 0, 0, z.stride(0), 0, f.stride(0))
        with _lib.on_device(z):
            _lib.check(_lib.lib().delrec_gated_step(
                ctypes.byref(s), z.data_ptr(), f.data_ptr(), _lib.addr(state), _lib.addr(active), h.data_ptr(),
                nxt.data_ptr(), _lib.stream_ptr(z.device)), "delrec_gated_step")
    return h, nxt
