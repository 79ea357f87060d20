"""Losses of a projection onto a large vocabulary that never form its logits: beside
``linear.readout_time_sum``, which serves a loss per sequence, these serve a loss per position.

    z_m = x_m weight^T + bias
    linear_cross_entropy     loss_m = logsumexp(z_m) - z_m[target_m]
    linear_distill           loss_m = tau^2 KL(softmax(t_m / tau) || softmax(z_m / tau)), where a
                             teacher's logits t_m are kept at K indices only

The (positions, vocabulary) logits live tile by tile in tensor memory; the backward pass forms
their gradient for a piece of the vocabulary at a time, as the operand of the products for dx and
dweight.  x, weight and bias are of one type, float32, bfloat16 or float16; sums are float32, and
float32 operands keep float32 accuracy (three bf16 pieces each).  In a 16-bit type, where there are
more than 512 positions, the logits' gradient is rounded to it once before the two products: the
gradients are then off by up to 1.4 times what their own rounding makes.  ``split=True`` keeps it in
two pieces, as few positions do: no more off than from a float32 one, for half to four fifths of the
training pass's time again.  CUDA tensors only.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
# An exponent z log2(e) / temperature is off by 2^-24 of itself: past 2^31 its power of two is no float any more.  The
# loss is good to some temperature^2 2^-20.
MIN_TEMPERATURE, MAX_TEMPERATURE = 1e-6, 1e6
MAX_FEATURES, MAX_KEPT, MAX_POSITIONS, MAX_VOCABULARY = 8192, 1024, 1 << 24, 1 << 30


def _struct(x, w, K, distill, reduction, lengths, index, logits, tau, ignore, split):
    T, B, D = x.shape
    wide = lambda t: 1 if t is not None and t.dtype == torch.int64 else 0   # noqa: E731
    return _lib.Vocab(T, B, D, w.shape[0], K, _lib.SEQ_DTYPES[x.dtype], distill, reduction, wide(lengths), wide(index),
                      _lib.SEQ_DTYPES[logits.dtype] if logits is not None else 0,
                      1 if w.data_ptr() % 16 == 0 else 0, tau, split, ignore, x.stride(0), x.stride(1))


def _forward(x, w, bias, index, logits, lengths, meta):
    """(loss, what the backward pass takes over)"""
    distill, reduction, tau, ignore, split = meta
    T, B, _ = x.shape
    dev = x.device
    out = torch.empty((T, B) if reduction == 0 else (), device=dev)
    if not (T and B):
        return out.zero_(), None
    s = _struct(x, w, index.shape[-1] if distill else 1, distill, reduction, lengths, index, logits, tau, ignore,
                split)
    lib, ref = _lib.lib(), ctypes.byref(s)
    nkeep, nbytes = lib.delrec_vocab_loss_keep(ref), lib.delrec_vocab_loss_forward_workspace(ref)
    keep, ws = _lib.scratch(nkeep, dev), _lib.scratch(nbytes, dev)
    A = _lib.addr
    _lib.launch("delrec_vocab_loss_forward", dev, ref, x.data_ptr(), w.data_ptr(), A(bias), index.data_ptr(), A(logits),
                A(lengths), out.data_ptr(), A(keep), nkeep, A(ws), nbytes)
    return out, keep


class VocabLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, index, logits, lengths, meta):
        ctx.set_materialize_grads(False)
        out, keep = _forward(x, w, bias, index, logits, lengths, meta)
        ctx.save_for_backward(x, w, bias, keep)
        ctx.meta = meta
        ctx.kept = index.shape[-1] if meta[0] else 1
        return out

    @staticmethod
    def backward(ctx, g):
        # the decorator's bookkeeping is wanted only where a second derivative could be
        return (_once if torch.is_grad_enabled() else _backward)(ctx, g)


def _backward(ctx, g):
    if g is None:
        return (None,) * 7
    x, w, bias, keep = ctx.saved_tensors
    distill, reduction, tau, ignore, split = ctx.meta
    need = ctx.needs_input_grad
    dev = x.device
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[0] else None
    dw = torch.empty_like(w) if need[1] else None
    db = torch.empty_like(bias) if bias is not None and need[2] else None
    if keep is not None:
        s = _struct(x, w, ctx.kept, distill, reduction, None, None, None, tau, ignore, split)
        lib, ref = _lib.lib(), ctypes.byref(s)
        nbytes = lib.delrec_vocab_loss_backward_workspace(ref)
        ws = _lib.scratch(nbytes, dev)
        A = _lib.addr
        g = g.contiguous()
        _lib.launch("delrec_vocab_loss_backward", dev, ref, x.data_ptr(), w.data_ptr(), A(bias), g.data_ptr(), A(keep),
                    keep.numel(), A(dx), A(dw), A(db), A(ws), nbytes)
    else:
        for t in (dw, db):
            if t is not None:
                t.zero_()
    return dx, dw, db, None, None, None, None


_once = once_differentiable(_backward)


def _check(x, weight, bias, reduction, lengths):
    """The leading shape of x; raises where the arguments do not fit one another."""
    _lib.require_sequence(x)
    shape, dtype, dev = x.shape, x.dtype, x.device
    if len(shape) < 2:
        raise RuntimeError(f"delrec_b200: x must be (T, B, D) or (.., D), got {tuple(shape)}")
    D = shape[-1]
    wshape = weight.shape
    if len(wshape) != 2 or wshape[1] != D or weight.dtype != dtype or weight.device != dev:
        raise RuntimeError(f"delrec_b200: weight must be (V, {D}) {dtype} on {dev}")
    V = wshape[0]
    if not 1 <= D <= MAX_FEATURES or not 1 <= V <= MAX_VOCABULARY:
        raise RuntimeError(f"delrec_b200: 1 to {MAX_FEATURES} features and a vocabulary of 1 to {MAX_VOCABULARY}, got "
                           f"{D} and {V}")
    if bias is not None and (bias.shape != (V,) or bias.dtype != dtype or bias.device != dev):
        raise RuntimeError(f"delrec_b200: bias must be ({V},) {dtype} on {dev}")
    if reduction not in REDUCTIONS:
        raise RuntimeError(f"delrec_b200: reduction must be one of {sorted(REDUCTIONS)}, got {reduction!r}")
    if shape[:-1].numel() > MAX_POSITIONS:
        raise RuntimeError(f"delrec_b200: at most {MAX_POSITIONS} positions, got {shape[:-1].numel()}")
    if lengths is not None:
        if len(shape) != 3:
            raise RuntimeError(f"delrec_b200: lengths are for x (T, B, D), got {tuple(shape)}")
        _lib.require_lengths(lengths, shape[1], dev)
    return shape[:-1]


def _run(x, w, bias, index, logits, lengths, meta, lead):
    if len(lead) == 1:
        x = x.unsqueeze(1)
    elif len(lead) > 2:
        x = x.reshape(-1, 1, x.shape[-1])
    x = _lib.rows(x)
    w = w.contiguous()
    bias = None if bias is None else bias.contiguous()
    index = index.contiguous()
    logits = None if logits is None else logits.detach().contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, bias)):
        out = VocabLoss.apply(x, w, bias, index, logits, lengths, meta)
    else:
        if getattr(forward_ad, "_current_level", 0) >= 0:
            _lib.refuse_tangents(x, w, bias, logits)
        out = _forward(x, w, bias, index, logits, lengths, meta)[0]
    return out.view(lead) if meta[1] == 0 else out


def linear_cross_entropy(x, weight, target, bias=None, *, ignore_index=-100, reduction="mean", lengths=None,
                         split=False):
    """Softmax cross entropy of x weight^T + bias against ``target``, in float32.

    x (T,B,D) or (.., D), weight (V,D), bias (V); target int32 / int64 of x's leading shape.  Positions
    whose target is ``ignore_index`` do not count: loss 0, gradient 0; nor do positions at or past
    ``lengths`` (B,) int32 / int64 (x (T,B,D)), where neither x nor target is read.  ``reduction``:
    "mean" over the positions that count (0 where none does), "sum", or "none" (losses of the leading
    shape).  Any other target outside the vocabulary makes its loss, and the gradients, NaN and sets a
    bit of ``_lib.status()``.  Gradients reach x, weight and bias; ``split``: how they are rounded in a
    16-bit type (above)."""
    lead = _check(x, weight, bias, reduction, lengths)
    if target.shape != lead or target.dtype not in (torch.int32, torch.int64) or target.device != x.device:
        raise RuntimeError(f"delrec_b200: target must be int32 or int64 {tuple(lead)} on {x.device}")
    ignore = int(ignore_index)
    if not -(1 << 63) <= ignore < 1 << 63:
        raise RuntimeError(f"delrec_b200: ignore_index {ignore} is past 64 bits")
    return _run(x, weight, bias, target, None, lengths, (0, REDUCTIONS[reduction], 1.0, ignore, 1 if split else 0), lead)


def linear_distill(x, weight, indices, logits, bias=None, *, temperature=1.0, reduction="mean", lengths=None,
                   split=False):
    """Distillation of x weight^T + bias from a teacher's K kept logits a position, in float32.

    x, weight, bias, ``reduction``, ``lengths``, ``split`` as in ``linear_cross_entropy``.  indices (.., K) int32 /
    int64 and logits (.., K) float32, bfloat16 or float16, K from 1 to 1024: the teacher's distribution
    is p = softmax(logits / temperature) over them, the student's q = softmax(z / temperature) over the
    whole vocabulary, loss = temperature^2 sum_k p_k (log p_k - log q[indices_k]), temperature from
    1e-6 to 1e6.  An entry with a negative index or a logit of -inf is left out; a position that keeps
    none does not count.  An index that stands twice counts twice.  An index past the vocabulary makes its loss, and the gradients,
    NaN and sets a bit of ``_lib.status()``.  Gradients reach x, weight and bias, not the teacher."""
    lead = _check(x, weight, bias, reduction, lengths)
    ishape = indices.shape
    if len(ishape) != len(lead) + 1 or ishape[:-1] != lead or indices.dtype not in (torch.int32, torch.int64) \
            or indices.device != x.device:
        raise RuntimeError(f"delrec_b200: indices must be int32 or int64 {tuple(lead)} + (K,) on {x.device}")
    if not 1 <= ishape[-1] <= MAX_KEPT:
        raise RuntimeError(f"delrec_b200: 1 to {MAX_KEPT} kept logits, got {ishape[-1]}")
    if logits.shape != ishape or logits.dtype not in _lib.SEQ_DTYPES or logits.device != x.device:
        raise RuntimeError(f"delrec_b200: logits must be float32, bfloat16 or float16 {tuple(ishape)} on {x.device}")
    if torch.is_grad_enabled() and logits.requires_grad:
        raise RuntimeError("delrec_b200: no gradient passes to the teacher's logits; detach them")
    tau = float(temperature)
    if not MIN_TEMPERATURE <= tau <= MAX_TEMPERATURE:
        raise RuntimeError(f"delrec_b200: temperature must be from {MIN_TEMPERATURE} to {MAX_TEMPERATURE}, got {temperature}")
    return _run(x, weight, bias, indices, logits, lengths, (1, REDUCTIONS[reduction], tau, 0, 1 if split else 0),
                lead)
