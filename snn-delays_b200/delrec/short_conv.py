"""Short causal convolution over time-major sequences, one filter of K taps per channel: what a
recurrent layer with input-dependent decay (``gated``, ``selective``) puts in front of its scan.

    p_t = bias + sum_{j<K} weight[:, j] x_{t-K+1+j},    y_t = act(p_t)

weight[:, K-1] belongs to the step itself.  Unlike ``dcls.Dcls1d`` the filter is dense in time and
the window in front of a piece of a sequence is a state that can be handed on, so pieces and
single steps (``short_conv_step``) give the numbers of the whole sequence.  CUDA tensors of type
float32, bfloat16 or float16; weight and bias are float32.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib

ACTS = {"none": 0, "silu": 1}
MAX_TAPS = 8


def _struct(dims, K, dtype, act, kind, *tensors):
    st = []
    for t in tensors:
        st += t.stride()[:2] if t is not None else (0, 0)
    return _lib.Conv(*dims, K, _lib.SEQ_DTYPES[dtype], act, kind, 0, *st)


def _forward(x, w, bias, state, lengths, resets, act):
    T, B, N = x.shape
    K = w.shape[1]
    dev = x.device
    y = _lib.empty_rows(x)
    new = torch.empty(K - 1, B, N, dtype=x.dtype, device=dev)
    if T and B and N:
        kind = 1 if lengths is not None and lengths.dtype == torch.int64 else 0
        s = _struct((T, B, N), K, x.dtype, act, kind, x, y)
        A = _lib.addr
        _lib.launch("delrec_short_conv_forward", dev, ctypes.byref(s), x.data_ptr(), w.data_ptr(), A(bias), A(state),
                    A(lengths), A(resets), y.data_ptr(), new.data_ptr() if K > 1 else None)
    elif state is not None:
        new.copy_(state)
    else:
        new.zero_()
    return y, new


class ShortConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, state, lengths, resets, act):
        ctx.set_materialize_grads(False)
        y, new = _forward(x, w, bias, state, lengths, resets, act)
        ctx.save_for_backward(x, w, bias, state, lengths, resets)
        ctx.act = act
        return y, new

    @staticmethod
    def backward(ctx, *grads):
        # the decorator's bookkeeping is wanted only where a second derivative could be
        return (_once if torch.is_grad_enabled() else _backward)(ctx, *grads)


def _backward(ctx, gy, gs):
    if gy is None and gs is None:
        return (None,) * 7
    x, w, bias, state, lengths, resets = ctx.saved_tensors
    T, B, N = x.shape
    K = w.shape[1]
    need = ctx.needs_input_grad
    dev = x.device
    dx = _lib.empty_rows(x) if need[0] else None
    dw = torch.empty(N, K, device=dev) if need[1] else None
    db = torch.empty(N, device=dev) if need[2] and bias is not None else None
    ds = torch.empty(K - 1, B, N, dtype=x.dtype, device=dev) if need[3] and state is not None else None
    if T and B and N:
        if gy is not None:
            gy = _lib.rows(gy)
        if gs is not None:
            gs = gs.contiguous()
        kind = 1 if lengths is not None and lengths.dtype == torch.int64 else 0
        s = _struct((T, B, N), K, x.dtype, ctx.act, kind, x, None, gy, dx)
        ws, nbytes = None, 0
        if dw is not None or db is not None:
            nbytes = _lib.lib().delrec_short_conv_backward_workspace(ctypes.byref(s))
            ws = _lib.scratch(nbytes, dev)
        A = _lib.addr
        _lib.launch("delrec_short_conv_backward", dev, ctypes.byref(s), x.data_ptr(), w.data_ptr(), A(bias), A(state),
                    A(lengths), A(resets), A(gy), A(gs) if K > 1 else None, A(dx), A(ds) if K > 1 else None, A(dw),
                    A(db), A(ws), nbytes)
    else:
        for t in (dw, db):
            if t is not None:
                t.zero_()
        if ds is not None:
            ds = gs.clone() if gs is not None else ds.zero_()
    return dx, dw, db, ds, None, None, None


_once = once_differentiable(_backward)


def _check(x, weight, bias, state, act, dims, layout):
    _lib.require_sequence(x)
    shape, dev = x.shape, x.device
    if len(shape) != dims:
        raise RuntimeError(f"delrec_b200: x must be {layout}, got {tuple(shape)}")
    _lib.require_sizes(*shape)
    if act not in ACTS:
        raise RuntimeError(f"delrec_b200: act must be one of {sorted(ACTS)}, got {act!r}")
    N = shape[-1]
    wshape = weight.shape
    if len(wshape) != 2 or wshape[0] != N or not 1 <= wshape[1] <= MAX_TAPS:
        raise RuntimeError(f"delrec_b200: weight must be ({N}, 1 to {MAX_TAPS} taps), got {tuple(wshape)}")
    if bias is not None and bias.shape != (N,):
        raise RuntimeError(f"delrec_b200: bias must be ({N},), got {tuple(bias.shape)}")
    for t in (weight, bias):
        if t is not None and (t.dtype != torch.float32 or t.device != dev):
            raise RuntimeError(f"delrec_b200: weight and bias must be float32 on {dev}")
    if state is not None:
        want = (wshape[1] - 1, shape[-2], N)
        if state.shape != want or state.dtype != x.dtype or state.device != dev:
            raise RuntimeError(f"delrec_b200: state must be {want} {x.dtype} on {dev}")
    return wshape[1]


def short_conv(x, weight, bias=None, state=None, *, act="silu", lengths=None, resets=None):
    """Convolve x (T,B,N) with weight (N,K), K from 1 to 8 -> (y (T,B,N), new state (K-1,B,N)).

    ``act``: "silu" or "none".  ``state`` (K-1,B,N), of x's type, holds the K-1 inputs before the
    first step, oldest first (None: zeros); the new state holds the last K-1 of each sequence.
    ``lengths`` (B,) int32 / int64: sequence b has lengths[b] steps; later positions are not
    read, their y and gradients are 0.  ``resets`` (T,B) bool: True drops the inputs before that step
    (sequences packed one after another), also from the new state.  Strides of T and B are free; a
    strided channel dimension is copied.  Gradients reach x, weight, bias and state."""
    _check(x, weight, bias, state, act, 3, "(T, B, N)")
    T, B, _ = x.shape
    if lengths is not None:
        _lib.require_lengths(lengths, B, x.device)
    resets = _lib.require_resets(resets, T, B, x.device)
    x, w = _lib.rows(x), weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    state = None if state is None else state.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, bias, state)):
        return ShortConvFn.apply(x, w, bias, state, lengths, resets, ACTS[act])
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _lib.refuse_tangents(x, w, bias, state)
    return _forward(x, w, bias, state, lengths, resets, ACTS[act])


def short_conv_step(x, weight, bias=None, state=None, *, act="silu", active=None, out=None):
    """One time step: x (B,N), state (K-1,B,N) of x's type (None: zeros) -> (y (B,N), next state).

    ``out`` receives the next state and may be ``state`` itself (updated in place), but no tensor
    that requires a gradient and none that overlaps it otherwise; None allocates it.  ``active``
    (B,) bool: a row with False keeps its state and gives y = 0.  No gradient passes; train with
    ``short_conv``."""
    K = _check(x, weight, bias, state, act, 2, "(B, N)")
    B, N = x.shape
    dev = x.device
    want = (K - 1, B, N)
    if out is not None:
        if out.shape != want or out.dtype != x.dtype or out.device != dev or not out.is_contiguous():
            raise RuntimeError(f"delrec_b200: out must be contiguous {want} {x.dtype} on {dev}")
        if torch.is_grad_enabled() and out.requires_grad:
            raise RuntimeError("delrec_b200: out must not require a gradient (no gradient passes)")
    active = _lib.require_active(active, B, dev)
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _lib.refuse_tangents(x, weight, bias, state)
    x, w = _lib.rows(x), weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    state = None if state is None else state.contiguous()
    y = torch.empty(B, N, device=dev, dtype=x.dtype)
    nxt = torch.empty(want, device=dev, dtype=x.dtype) if out is None else out
    if B and N:
        s = _lib.Conv(1, B, N, K, _lib.SEQ_DTYPES[x.dtype], ACTS[act], 2, 0, 0, x.stride(0), 0, N)
        A = _lib.addr
        _lib.launch("delrec_short_conv_forward", dev, ctypes.byref(s), x.data_ptr(), w.data_ptr(), A(bias),
                    A(state) if K > 1 else None, A(active), None, y.data_ptr(), nxt.data_ptr() if K > 1 else None)
    if out is not None:
        increment_version(out)       # who saved the old state for a gradient learns of it
    return y, nxt
