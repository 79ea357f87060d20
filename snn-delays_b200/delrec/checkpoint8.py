"""Activations kept in 8 bits between the forward and the backward pass.

``pack8`` stores rows of channels as int8 with one power-of-two scale per group of 32
consecutive channels (8.25 bits a value), ``unpack8`` restores them.  A value is kept to
within half a step, 2^-7 to 2^-8 of its group's largest magnitude; 0 / 1 spike trains,
infinities and NaN come back exactly.  ``linear.Linear(checkpoint8=True)`` and
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
    x = x.detach().contiguous()
    p = empty8(x.shape, x.dtype, x.device)
    if x.numel():
        with _lib.on_device(x):
            _lib.check(_lib.lib().delrec_pack8(x.numel() // x.shape[-1], x.shape[-1], code, x.data_ptr(),
                                               p.q.data_ptr(), p.e.data_ptr(), _lib.stream_ptr(x.device)),
                       "delrec_pack8")
    return p


def unpack8(packed: Packed8, dtype=None):
    """The tensor that ``packed`` stands for, in its own dtype or the given one."""
    q, e = packed.q, packed.e
    dtype = packed.dtype if dtype is None else dtype
    if dtype not in _lib.SEQ_DTYPES:
        raise RuntimeError(f"delrec_b200 expects float32, bfloat16 or float16, got {dtype}")
    if not (q.is_cuda and e.device == q.device):
        raise RuntimeError("delrec_b200 runs on CUDA tensors only (there is no CPU path)")
    if (q.dtype, e.dtype) != (torch.int8, torch.uint8) or q.dim() == 0 \
            or e.shape != (*q.shape[:-1], -(-q.shape[-1] // GROUP)):
        raise RuntimeError("delrec_b200: not a Packed8 (int8 (..., N) with uint8 (..., ceil(N / 32)))")
    q, e = q.contiguous(), e.contiguous()
    x = torch.empty(q.shape, dtype=dtype, device=q.device)
    if x.numel():
        with _lib.on_device(q):
            _lib.check(_lib.lib().delrec_unpack8(q.numel() // q.shape[-1], q.shape[-1], _lib.SEQ_DTYPES[dtype],
                                                 q.data_ptr(), e.data_ptr(), x.data_ptr(),
                                                 _lib.stream_ptr(q.device)), "delrec_unpack8")
    return x
