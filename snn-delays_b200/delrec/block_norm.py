"""RMS norms before and after a block, fused with its gate, residual scale and residual sum.

    block_norm(x, weight)       x / rms(x) * weight                       (before the first block)
    block_join(x, y, weight, gate, scale, next_weight)
        x' = x + scale * act(gate) * (y / rms(y) * weight)                (after a block)
        n  = x' / rms(x') * next_weight                                   (before the next one)

with rms(v) = sqrt(mean v^2 + eps) over the channels of a position.  Unlike
``neuron.BatchNorm1d`` a position's norm depends on no other one, so padded batches and
streaming steps give the same numbers as whole sequences.  x, y and gate are (T,B,N)
float32, bfloat16 or float16; the weights are (N,) float32.  CUDA tensors only.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib

GATES = {"none": 0, "sigmoid": 1, "silu": 2}


def _strides(b, **tensors):
    for name, t in tensors.items():
        if t is not None:
            setattr(b, name + "_t", t.stride(0))
            setattr(b, name + "_b", t.stride(1))


class BlockNormFn(torch.autograd.Function):
    """(x, y, gate, weight, scale, next_weight) -> (x', n); n alone without y, x' alone
    without ``has_next``."""

    @staticmethod
    def forward(ctx, x, y, u, w, scale, nw, lengths, kind, eps, has_next):
        ctx.set_materialize_grads(False)
        x, y, u = (None if t is None else _lib.rows(t.detach()) for t in (x, y, u))
        w, scale, nw = (None if t is None else t.detach().contiguous() for t in (w, scale, nw))
        T, B, N = x.shape
        dev = x.device
        out = _lib.empty_rows(x) if y is not None else None
        n = _lib.empty_rows(x) if has_next else None
        train = any(ctx.needs_input_grad[:6])
        ry = torch.empty(T, B, device=dev) if train and y is not None else None
        rx = torch.empty(T, B, device=dev) if train and has_next else None
        b = _lib.Block(T, B, N, _lib.SEQ_DTYPES[x.dtype], kind,
                       int(lengths is not None and lengths.dtype == torch.int64), eps, 0)
        _strides(b, x=x, y=y, u=u, o=out, n=n)
        if T and B and N:
            A = _lib.addr
            with _lib.on_device(x):
                _lib.check(_lib.lib().delrec_block_norm_forward(
                    ctypes.byref(b), A(x), A(y), A(u), A(w), A(scale), A(nw), A(lengths), A(out), A(n), A(ry),
                    A(rx), _lib.stream_ptr(dev)), "delrec_block_norm_forward")
        if train:
            ctx.save_for_backward(x if has_next else None, y, u, w, scale, nw, lengths, ry, rx)
            ctx.block, ctx.shape, ctx.dtype, ctx.has_next = b, (T, B, N), x.dtype, has_next
        outs = tuple(t for t in (out, n) if t is not None)
        return outs if len(outs) > 1 else outs[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        x, y, u, w, scale, nw, lengths, ry, rx = ctx.saved_tensors
        T, B, N = ctx.shape
        gx = grads[0] if y is not None else None
        gn = grads[-1] if ctx.has_next else None
        if gx is None and gn is None:
            return (None,) * 10
        gx, gn = (None if g is None else _lib.rows(g) for g in (gx, gn))
        dev = (gx if gx is not None else gn).device
        need = ctx.needs_input_grad
        like = x if x is not None else y
        new = lambda want: _lib.empty_rows(like) if want else None   # noqa: E731
        vec = lambda want: torch.empty(N, device=dev) if want else None   # noqa: E731
        dx, dy, du = new(need[0]), new(need[1]), new(need[2])
        dw, ds, dn = vec(need[3]), vec(need[4]), vec(need[5])
        if not (T and B and N):
            for t in (dw, ds, dn):
                if t is not None:
                    t.zero_()
            return dx, dy, du, dw, ds, dn, None, None, None, None
        b = _lib.Block.from_buffer_copy(ctx.block)
        _strides(b, gx=gx, gn=gn, dx=dx, dy=dy, du=du)
        lib, A = _lib.lib(), _lib.addr
        sums = any(t is not None for t in (dw, ds, dn))
        nbytes = lib.delrec_block_norm_backward_workspace(ctypes.byref(b)) if sums else 0
        ws = _lib.scratch(nbytes, dev)
        with _lib.on_device(like):
            _lib.check(lib.delrec_block_norm_backward(
                ctypes.byref(b), A(x), A(y), A(u), A(w), A(scale), A(nw), A(lengths), A(ry), A(rx), A(gx), A(gn),
                A(dx), A(dy), A(du), A(dw), A(ds), A(dn), A(ws), nbytes, _lib.stream_ptr(dev)),
                "delrec_block_norm_backward")
        return dx, dy, du, dw, ds, dn, None, None, None, None


def _check(x, others, weights, lengths, eps):
    _lib.require_sequence(x, *(t for t in others if t is not None))
    if x.dim() != 3:
        raise RuntimeError(f"delrec_b200: x must be (T, B, N), got {tuple(x.shape)}")
    for t in others:
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype or t.device != x.device):
            raise RuntimeError("delrec_b200: x, y and gate must share shape, dtype and device")
    for w in weights:
        if w is not None and (w.shape != (x.shape[-1],) or w.dtype != torch.float32 or w.device != x.device):
            raise RuntimeError(f"delrec_b200: weights must be ({x.shape[-1]},) float32 on {x.device}")
    if not eps > 0:
        raise RuntimeError("delrec_b200: eps must be positive")
    if lengths is not None:
        _lib.require_lengths(lengths, x.shape[1], x.device)


def block_norm(x, weight=None, *, eps=1e-5, lengths=None):
    """x (T,B,N) -> x / rms(x) * weight.  ``lengths`` (B,): positions t >= lengths[b] are not
    read, their outputs and gradients are 0.  Strides of T and B are free."""
    _check(x, (), (weight,), lengths, eps)
    return BlockNormFn.apply(x, None, None, None, None, weight, lengths, 0, eps, True)


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
    r = BlockNormFn.apply(x, y, gate if kind else None, weight, scale, next_weight, lengths, kind, eps, has_next)
    return r if has_next else (r, None)
