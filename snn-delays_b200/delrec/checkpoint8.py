"""Activations kept in 8 bits between the forward and the backward pass.

``pack8`` stores rows of channels as int8 with one power-of-two scale per group of 32
consecutive channels (8.25 bits a value), ``unpack8`` restores them.  A value is kept to
within half a step, 1/252 to 1/126 of its group's largest magnitude m where 2^-120 <= m <
63.5 * 2^122; within 2^-127 where m is smaller, within 2^122 where it is larger.  0 / 1 spike
trains, infinities and NaN come back exactly.  ``linear.Linear(checkpoint8=True)`` and
``gated.gated_scan(checkpoint8=True)`` keep what they save for the backward pass this way.
CUDA tensors only.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

GROUP = 32


class Packed8(NamedTuple):
    """x (..., N) in 8 bits: x = q * 2^(e - 127), e shared by 32 channels."""
    q: torch.Tensor        # int8 (..., N); 127: +inf, -127: -inf, -128: NaN
    e: torch.Tensor        # uint8 (..., ceil(N / 32))
    dtype: torch.dtype     # of the packed tensor

    @property
    def nbytes(self):
        return self.q.numel() + self.e.numel()


def empty8(shape, dtype, device):
    """The buffers of a Packed8 of the given shape."""
    return Packed8(torch.empty(shape, dtype=torch.int8, device=device),
                   torch.empty(*shape[:-1], -(-shape[-1] // GROUP), dtype=torch.uint8, device=device), dtype)


def pack8(x) -> Packed8:
    """x (..., N) float32, bfloat16 or float16 in 8 bits (no gradient passes)."""
    code = _lib.require_sequence(x)
    if x.dim() == 0:
        raise RuntimeError("delrec_b200: pack8 expects at least one dimension")
    _lib.require_sizes(x.shape[-1])
    x = x.contiguous()
    shape, device = x.shape, x.device
    p = empty8(shape, x.dtype, device)
    n = x.numel()
    if n:
        _lib.launch("delrec_pack8", device, n // shape[-1], shape[-1], code, x.data_ptr(), p.q.data_ptr(),
                    p.e.data_ptr())
    return p


def unpack8(packed: Packed8, dtype=None):
    """The tensor that ``packed`` stands for, in its own dtype or the given one (float16
    saturates at its largest value)."""
    q, e, own = packed
    code = _lib.SEQ_DTYPES.get(dtype or own)
    if code is None:
        raise RuntimeError(f"delrec_b200 expects float32, bfloat16 or float16, got {dtype or own}")
    device = q.device
    if not q.is_cuda or e.device != device:
        raise RuntimeError("delrec_b200 runs on CUDA tensors only (there is no CPU path)")
    shape = q.shape
    if q.dtype != torch.int8 or e.dtype != torch.uint8 or q.dim() == 0 \
            or e.shape != (*shape[:-1], -(-shape[-1] // GROUP)):
        raise RuntimeError("delrec_b200: not a Packed8 (int8 (..., N) with uint8 (..., ceil(N / 32)))")
    _lib.require_sizes(shape[-1])
    q, e = q.contiguous(), e.contiguous()
    x = torch.empty(shape, dtype=dtype or own, device=device)
    n = x.numel()
    if n:
        _lib.launch("delrec_unpack8", device, n // shape[-1], shape[-1], code, q.data_ptr(), e.data_ptr(),
                    x.data_ptr())
    return x
