"""RMS norms before and after a block, fused with its gate, residual scale and residual sum.

    block_norm(x, weight)       x / rms(x) * weight                       (before the first block)
    block_join(x, y, weight, gate, scale, next_weight)
        x' = x + scale * act(gate) * (y / rms(y) * weight)                (after a block)
        n  = x' / rms(x') * next_weight                                   (before the next one)

with rms(v) = sqrt(mean v^2 + eps) over the channels of a position.  Unlike
``neuron.BatchNorm1d`` a position's norm depends on no other one, so padded batches and
streaming steps give the same numbers as whole sequences.  The sum of a position's squares
is float32 and has to stay below 3.4e38.  x, y and gate are (T,B,N)
float32, bfloat16 or float16; the weights are (N,) float32.  CUDA tensors only.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

GATES = {"none": 0, "sigmoid": 1, "silu": 2}


def _strides(*tensors):
    r = []
    for t in tensors:
        r += t.stride()[:2] if t is not None else (0, 0)
    return r


def _wide(lengths):
    return 1 if lengths is not None and lengths.dtype == torch.int64 else 0


def _forward(x, y, u, w, scale, nw, lengths, kind, eps, has_next, train):
    """(x', n, 1/rms of y, 1/rms of x'), None where there is none: one launch."""
    T, B, N = x.shape
    dev = x.device
    out = _lib.empty_rows(x) if y is not None else None
    n = _lib.empty_rows(x) if has_next else None
    ry = torch.empty(T, B, device=dev) if train and y is not None else None
    rx = torch.empty(T, B, device=dev) if train and has_next else None
    if T and B and N:
        b = _lib.Block(T, B, N, _lib.SEQ_DTYPES[x.dtype], kind, _wide(lengths), eps, 0, *_strides(x, y, u, out, n))
        A = _lib.addr
        _lib.launch("delrec_block_norm_forward", dev, ctypes.byref(b), x.data_ptr(), A(y), A(u), A(w), A(scale), A(nw),
                    A(lengths), A(out), A(n), A(ry), A(rx))
    return out, n, ry, rx


class BlockNormFn(torch.autograd.Function):
    """(x, y, gate, weight, scale, next_weight) -> (x', n); n alone without y, x' alone
    without ``has_next``."""

    @staticmethod
    def forward(ctx, x, y, u, w, scale, nw, lengths, kind, eps, has_next):
        ctx.set_materialize_grads(False)
        out, n, ry, rx = _forward(x, y, u, w, scale, nw, lengths, kind, eps, has_next, True)
        ctx.save_for_backward(x if has_next else None, y, u, w, scale, nw, lengths, ry, rx)
        ctx.meta = x.shape, x.dtype, kind, eps, has_next
        if out is None:
            return n
        return (out, n) if has_next else out

    @staticmethod
    def backward(ctx, *grads):
        # the decorator's bookkeeping is wanted only where a second derivative could be
        return (_once if torch.is_grad_enabled() else _backward)(ctx, *grads)


def _backward(ctx, *grads):
    x, y, u, w, scale, nw, lengths, ry, rx = ctx.saved_tensors
    (T, B, N), dtype, kind, eps, has_next = ctx.meta
    gx = grads[0] if y is not None else None
    gn = grads[-1] if has_next else None
    if gx is None and gn is None:
        return (None,) * 10
    if gx is not None:
        gx = _lib.rows(gx)
    if gn is not None:
        gn = _lib.rows(gn)
    need = ctx.needs_input_grad
    like = x if x is not None else y
    dev = like.device
    dx = _lib.empty_rows(like) if need[0] else None
    dy = _lib.empty_rows(like) if need[1] else None
    du = _lib.empty_rows(like) if need[2] else None
    dw = torch.empty(N, device=dev) if need[3] else None
    ds = torch.empty(N, device=dev) if need[4] else None
    dn = torch.empty(N, device=dev) if need[5] else None
    if T and B and N:
        b = _lib.Block(T, B, N, _lib.SEQ_DTYPES[dtype], kind, _wide(lengths), eps, 0,
                       *_strides(x, y, u, None, None, gx, gn, dx, dy, du))
        ws, nbytes = None, 0
        if dw is not None or ds is not None or dn is not None:
            nbytes = _lib.lib().delrec_block_norm_backward_workspace(ctypes.byref(b))
            ws = _lib.scratch(nbytes, dev)
        A = _lib.addr
        _lib.launch("delrec_block_norm_backward", dev, ctypes.byref(b), A(x), A(y), A(u), A(w), A(scale), A(nw),
                    A(lengths), A(ry), A(rx), A(gx), A(gn), A(dx), A(dy), A(du), A(dw), A(ds), A(dn), A(ws), nbytes)
    else:
        for t in (dw, ds, dn):
            if t is not None:
                t.zero_()
    return dx, dy, du, dw, ds, dn, None, None, None, None


_once = once_differentiable(_backward)


def _run(x, y, u, w, scale, nw, lengths, kind, eps, has_next):
    """(x', n) through autograd where a gradient is wanted, else plainly."""
    args = [None if t is None else _lib.rows(t) for t in (x, y, u)]
    args += [None if t is None else t.contiguous() for t in (w, scale, nw)]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        r = BlockNormFn.apply(*args, lengths, kind, eps, has_next)
        if y is None:
            return None, r
        return r if has_next else (r, None)
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _lib.refuse_tangents(*args)
    return _forward(*args, lengths, kind, eps, has_next, False)[:2]


def _check(x, others, weights, lengths, eps):
    _lib.require_sequence(x)
    shape, dtype, device = x.shape, x.dtype, x.device
    if len(shape) != 3:
        raise RuntimeError(f"delrec_b200: x must be (T, B, N), got {tuple(shape)}")
    _lib.require_sizes(*shape)
    for t in others:
        if t is not None and (t.shape != shape or t.dtype != dtype or t.device != device):
            raise RuntimeError("delrec_b200: x, y and gate must share shape, dtype and device")
    for w in weights:
        if w is not None and (w.shape != shape[2:] or w.dtype != torch.float32 or w.device != device):
            raise RuntimeError(f"delrec_b200: weights must be ({shape[2]},) float32 on {device}")
    if not eps > 0:
        raise RuntimeError("delrec_b200: eps must be positive")
    if lengths is not None:
        _lib.require_lengths(lengths, shape[1], device)


def block_norm(x, weight=None, *, eps=1e-5, lengths=None):
    """x (T,B,N) -> x / rms(x) * weight.  ``lengths`` (B,): positions t >= lengths[b] are not
    read, their outputs and gradients are 0.  Strides of T and B are free."""
    _check(x, (), (weight,), lengths, eps)
    return _run(x, None, None, None, None, weight, lengths, 0, eps, True)[1]


def block_join(x, y, weight=None, *, gate=None, gate_act="sigmoid", scale=None, next_weight=None,
               next_norm=None, eps=1e-5, lengths=None):
    """Join a block's output y to the residual stream x -> (x', n).

    x' = x + scale * act(gate) * (y / rms(y) * weight), act by ``gate_act`` ("sigmoid",
    "silu", "none"; no ``gate``: 1); ``scale`` is the per-channel residual scale (N,).
    n = x' / rms(x') * next_weight feeds the next block; it is formed from the unrounded x'.
    It is None unless ``next_weight`` is given or ``next_norm=True`` (a norm without weight).
    ``lengths`` as in ``block_norm``.  Gradients reach every tensor argument."""
    if gate_act not in GATES:
        raise RuntimeError(f"delrec_b200: gate_act must be one of {sorted(GATES)}, got {gate_act!r}")
    _check(x, (y, gate), (weight, scale, next_weight), lengths, eps)
    if y is None:
        raise RuntimeError("delrec_b200: block_join needs the block's output y")
    has_next = next_weight is not None if next_norm is None else bool(next_norm)
    if next_weight is not None and not has_next:
        raise RuntimeError("delrec_b200: next_weight without a next norm")
    kind = GATES[gate_act] if gate is not None else 0
    return _run(x, y, gate if kind else None, weight, scale, next_weight, lengths, kind, eps, has_next)
