"""Selective state space scan over time-major sequences: a recurrence like ``gated.gated_scan``
with S states to a channel, whose step size, input and output weights depend on the input.

    delta_t = softplus(dt_t + dt_bias)
    h_t[n,s] = exp(delta_t[n] A[n,s]) h_{t-1}[n,s] + delta_t[n] B_t[g,s] x_t[n]
    y_t[n] = (sum_s C_t[g,s] h_t[n,s] + D[n] x_t[n]) silu(gate_t[n])

``selective_scan`` runs whole sequences and is differentiable, ``selective_step`` one time step for
streaming.  x, dt, gate are (T,B,N), B and C (T,B,S), or (T,B,G,S) where group g serves the N / G
channels from g N / G on, of type float32, bfloat16 or float16; A (N,S), D and dt_bias (N) and the
states are float32; S from 1 to 128.  CUDA tensors only.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib

SEGMENT = 8      # distance of the states kept for the backward pass
MAX_STATES = 128


def _struct(x, S, G, softplus, lengths, dims, gate, y, Bm, Cm, *tensors):
    st = []
    for t in (x, dims, gate, y, Bm, Cm) + tensors:
        st += t.stride()[:2] if t is not None else (0, 0)
    wide = 1 if lengths is not None and lengths.dtype == torch.int64 else 0
    return _lib.Selective(*x.shape, S, G, _lib.SEQ_DTYPES[x.dtype], 1 if softplus else 0, wide,
                          1 if lengths is not None else 0, 0, *st)


def _forward(x, dt, A, Bm, Cm, h0, D, gate, dt_bias, lengths, resets, softplus, train):
    """(y, hT, states kept for the backward pass or None)"""
    T, B, N = x.shape
    G, S = Bm.shape[2:]
    dev = x.device
    y = _lib.empty_rows(x)
    hT = torch.empty(B, N, S, device=dev)
    states = torch.empty(-(-T // SEGMENT), B, N, S, device=dev) if train else None
    if T and B and N:
        s = _struct(x, S, G, softplus, lengths, dt, gate, y, Bm, Cm)
        lib = _lib.lib()
        nbytes = lib.delrec_selective_forward_workspace(ctypes.byref(s))
        ws = _lib.scratch(nbytes, dev)
        P = _lib.addr
        _lib.launch("delrec_selective_forward", dev, ctypes.byref(s), x.data_ptr(), dt.data_ptr(), A.data_ptr(),
                    Bm.data_ptr(), Cm.data_ptr(), P(D), P(gate), P(dt_bias), P(h0), P(lengths), P(resets),
                    y.data_ptr(), hT.data_ptr(), P(states), P(ws), nbytes)
    elif h0 is not None:
        hT.copy_(h0)
    else:
        hT.zero_()
    return y, hT, states


class SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, Bm, Cm, h0, D, gate, dt_bias, lengths, resets, softplus):
        ctx.set_materialize_grads(False)
        y, hT, states = _forward(x, dt, A, Bm, Cm, h0, D, gate, dt_bias, lengths, resets, softplus, True)
        ctx.save_for_backward(x, dt, A, Bm, Cm, D, gate, dt_bias, lengths, resets, states)
        ctx.softplus = softplus
        return y, hT

    @staticmethod
    def backward(ctx, *grads):
        # the decorator's bookkeeping is wanted only where a second derivative could be
        return (_once if torch.is_grad_enabled() else _backward)(ctx, *grads)


def _backward(ctx, gy, ghT):
    if gy is None and ghT is None:
        return (None,) * 12
    x, dt, A, Bm, Cm, D, gate, dt_bias, lengths, resets, states = ctx.saved_tensors
    T, B, N = x.shape
    G, S = Bm.shape[2:]
    dev = x.device
    need = ctx.needs_input_grad
    new = lambda i, t, like=None: _lib.empty_rows(t) if need[i] and t is not None else None   # noqa: E731
    small = lambda i, t: torch.empty(t.shape, device=dev) if need[i] and t is not None else None   # noqa: E731
    dx, ddt, dgate = new(0, x), new(1, dt), new(7, gate)
    dA, dD, dbias = small(2, A), small(6, D), small(8, dt_bias)
    dB = torch.empty(Bm.shape, dtype=x.dtype, device=dev) if need[3] else None
    dC = torch.empty(Cm.shape, dtype=x.dtype, device=dev) if need[4] else None
    dh0 = torch.empty(B, N, S, device=dev) if need[5] else None
    if T and B and N:
        if gy is not None:
            gy = _lib.rows(gy)
        if ghT is not None:
            ghT = ghT.contiguous()
        s = _struct(x, S, G, ctx.softplus, lengths, dt, gate, None, Bm, Cm, gy, dx, ddt, dgate)
        s.no_bc = 1 if dB is None and dC is None else 0
        nbytes = _lib.lib().delrec_selective_backward_workspace(ctypes.byref(s))
        ws = _lib.scratch(nbytes, dev)
        P = _lib.addr
        _lib.launch("delrec_selective_backward", dev, ctypes.byref(s), x.data_ptr(), dt.data_ptr(), A.data_ptr(),
                    Bm.data_ptr(), Cm.data_ptr(), P(D), P(gate), P(dt_bias), P(lengths), P(resets), states.data_ptr(),
                    P(gy), P(ghT), P(dx), P(ddt), P(dA), P(dB), P(dC), P(dD), P(dgate), P(dbias), P(dh0), P(ws),
                    nbytes)
    else:
        for t in (dA, dD, dbias, dB, dC):
            if t is not None:
                t.zero_()
        if dh0 is not None:
            dh0 = ghT.clone() if ghT is not None else dh0.zero_()
    return dx, ddt, dA, dB, dC, dh0, dD, dgate, dbias, None, None, None


_once = once_differentiable(_backward)


def _check(x, dt, A, B, C, D, gate, dt_bias, state, name, dims):
    _lib.require_sequence(x)
    shape, dtype, dev = x.shape, x.dtype, x.device
    lead = "T, B" if dims == 3 else "B"
    if len(shape) != dims:
        raise RuntimeError(f"delrec_b200: x must be ({lead}, N), got {tuple(shape)}")
    _lib.require_sizes(*shape)
    N = shape[-1]
    for t in (dt, gate):
        if t is not None and (t.shape != shape or t.dtype != dtype or t.device != dev):
            raise RuntimeError("delrec_b200: x, dt and gate must share shape, dtype and device")
    ashape = A.shape
    if len(ashape) != 2 or ashape[0] != N or not 1 <= ashape[1] <= MAX_STATES:
        raise RuntimeError(f"delrec_b200: A must be ({N}, 1 to {MAX_STATES} states), got {tuple(ashape)}")
    S = ashape[1]
    bshape = B.shape
    if len(bshape) not in (dims, dims + 1) or bshape[:dims - 1] != shape[:-1] or bshape[-1] != S or C.shape != bshape:
        raise RuntimeError(f"delrec_b200: B and C must be ({lead}, {S}) or ({lead}, G, {S}), got {tuple(bshape)} and "
                           f"{tuple(C.shape)}")
    for t in (B, C):
        if t.dtype != dtype or t.device != dev:
            raise RuntimeError("delrec_b200: x, B and C must share dtype and device")
    G = bshape[-2] if len(bshape) == dims + 1 else 1
    if G == 0 or N % G:
        raise RuntimeError(f"delrec_b200: the {G} groups of B and C must divide the {N} channels of x")
    for t, want, what in ((A, ashape, "A"), (D, (N,), "D"), (dt_bias, (N,), "dt_bias"),
                          (state, (shape[-2], N, S), name)):
        if t is not None and (t.shape != want or t.dtype != torch.float32 or t.device != dev):
            raise RuntimeError(f"delrec_b200: {what} must be {tuple(want)} float32 on {dev}")
    return G, S


def _groups(t, dims, G, S):
    """B or C as (.., G, S) with contiguous (G, S)."""
    if t.dim() == dims:
        t = t.unsqueeze(-2)
    ok = (S == 1 or t.stride(-1) == 1) and (G == 1 or t.stride(-2) == S)
    return t if ok else t.contiguous()


def selective_scan(x, dt, A, B, C, h0=None, *, D=None, gate=None, dt_bias=None, softplus=True, lengths=None,
                   resets=None):
    """Run the recurrence over x (T,B,N) -> (y (T,B,N), hT (B,N,S)).

    A is negative for a state that decays.  ``softplus=False`` takes dt + dt_bias as the step size
    itself.  ``h0`` (B,N,S) float32 is the state before the first step (None: 0), ``hT`` the state
    after the last.  ``D`` None: no skip term; ``gate`` None: 1; ``dt_bias`` None: 0.  ``lengths`` (B,) int32 /
    int64: sequence b has lengths[b] steps; later positions are not read, their y and gradients
    are 0, and hT is the state after the last step there is.  ``resets`` (T,B) bool: True drops the
    state before that step (sequences packed one after another).  A decay below 1.2e-38 counts as
    0, and A = -inf is one of 0 at every step whose delta is not 0.  Strides of T and B are free; a strided channel (or group and state) dimension is copied.

    Gradients reach x, dt, A, B, C, h0, D, gate and dt_bias.  For the backward pass the inputs are
    kept, and the float32 state before every 8th step.  Where B or C learns, sums over channels take
    twice (T,B,G,S) float32 while it runs, for each tile of 8 (S > 64) to 256 (S <= 4) channels
    of a group, but no more than those states take where that fills the GPU."""
    G, S = _check(x, dt, A, B, C, D, gate, dt_bias, h0, "h0", 3)
    T, Bs, _ = x.shape
    if lengths is not None:
        _lib.require_lengths(lengths, Bs, x.device)
    resets = _lib.require_resets(resets, T, Bs, x.device)
    c = lambda t: None if t is None else t.contiguous()   # noqa: E731
    args = (_lib.rows(x), _lib.rows(dt), A.contiguous(), _groups(B, 3, G, S), _groups(C, 3, G, S), c(h0), c(D),
            None if gate is None else _lib.rows(gate), c(dt_bias))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        return SelectiveScan.apply(*args, lengths, resets, bool(softplus))
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _lib.refuse_tangents(*args)
    return _forward(*args, lengths, resets, softplus, False)[:2]


def selective_step(x, dt, A, B, C, state=None, *, D=None, gate=None, dt_bias=None, softplus=True, active=None,
                   out=None):
    """One time step: x, dt, gate (B,N), B and C (B,S) or (B,G,S), state (B,N,S) float32 (None: 0)
    -> (y (B,N), next state).

    ``out`` receives the next state and may be ``state`` itself (updated in place), but no tensor
    that requires a gradient and none that overlaps it otherwise; None allocates it.  ``active``
    (B,) bool: a row with False keeps its state and gives y = 0.  No gradient passes; train with
    ``selective_scan``."""
    G, S = _check(x, dt, A, B, C, D, gate, dt_bias, state, "state", 2)
    Bs, N = x.shape
    dev = x.device
    if out is not None:
        if out.shape != (Bs, N, S) or out.dtype != torch.float32 or out.device != dev or not out.is_contiguous():
            raise RuntimeError(f"delrec_b200: out must be contiguous ({Bs}, {N}, {S}) float32 on {dev}")
        if torch.is_grad_enabled() and out.requires_grad:
            raise RuntimeError("delrec_b200: out must not require a gradient (no gradient passes)")
    active = _lib.require_active(active, Bs, dev)
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _lib.refuse_tangents(x, dt, A, B, C, state, D, gate, dt_bias)
    c = lambda t: None if t is None else t.contiguous()   # noqa: E731
    x, dt, gate = _lib.rows(x), _lib.rows(dt), None if gate is None else _lib.rows(gate)
    A, B, C, state, D, dt_bias = c(A), _groups(B, 2, G, S), _groups(C, 2, G, S), c(state), c(D), c(dt_bias)
    y = torch.empty(Bs, N, device=dev, dtype=x.dtype)
    nxt = torch.empty(Bs, N, S, device=dev) if out is None else out
    if Bs and N:
        s = _lib.Selective(1, Bs, N, S, G, _lib.SEQ_DTYPES[x.dtype], 1 if softplus else 0, 0, 0, 0, 0, x.stride(0),
                           0, dt.stride(0), 0, gate.stride(0) if gate is not None else 0, 0, N, 0, B.stride(0), 0,
                           C.stride(0))
        P = _lib.addr
        _lib.launch("delrec_selective_step", dev, ctypes.byref(s), x.data_ptr(), dt.data_ptr(), A.data_ptr(),
                    B.data_ptr(), C.data_ptr(), P(D), P(gate), P(dt_bias), P(state), P(active), y.data_ptr(),
                    nxt.data_ptr())
    if out is not None:
        increment_version(out)       # who saved the old state for a gradient learns of it
    return y, nxt
