"""Activation checkpoints in 8 bits.

`pack` turns activations into int8 with one power of two for each 128
neighbouring values of the last dimension (1 + 1/128 bytes a value), `unpack`
turns them back into the type they had.  The scale is the smallest power of
two 2^e with max|v| <= 127 2^e, so a value is off by at most 2^(e-1), less
than max|v| / 126 of its group, and unpacking itself rounds nothing in bf16 and
fp32.  A group that holds a NaN or an infinity unpacks to NaN.

At the ends of a type's range e is limited.  It is at least -126: a group with
max|v| below 2^-120 or so is off by up to 2^-127, which may be more than
max|v| / 126.  It is at most 9 in fp16 and 121 in bf16 and fp32, so that the
restored values are finite: beyond 127 2^e (65024 in fp16, 3.376e38) a value
comes back as that, off by less than 2^e.

`prefill.run_autograd(..., checkpoint="int8")` and
`recurrence.run_autograd(..., checkpoint="int8")` keep their inputs this way
between forward and backward.  No counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Sequence

import torch

from . import _native
from .recurrence import _TYPES, _call

GROUP = 128
MAX_TENSORS = 4  # of one launch; more take several


class Packed:
    """Tensors of one type in 8 bits: one buffer, and what was put into it."""

    __slots__ = ("buffer", "dtype", "shapes", "places")

    def __init__(self, buffer, dtype, shapes, places):
        # places: per tensor where its values and its scales start, rows, columns
        self.buffer, self.dtype, self.shapes, self.places = buffer, dtype, shapes, places

    def __len__(self):
        return len(self.shapes)

    def nbytes(self) -> int:
        return self.buffer.numel()

    def values(self, i: int) -> torch.Tensor:
        """The int8 values of tensor i, in its shape (a view of the buffer)."""
        shape, at = self.shapes[i], self.places[i][0]
        return self.buffer[at:at + _count(shape)].view(torch.int8).view(shape)

    def scales(self, i: int) -> torch.Tensor:
        """The exponent bytes E (scale 2^(E-127); 255: not finite) of tensor i,
        [..., ceil(last / 128)] uint8 (a view of the buffer)."""
        shape, at = self.shapes[i], self.places[i][1]
        shape = (*shape[:-1], -(-shape[-1] // GROUP))
        return self.buffer[at:at + _count(shape)].view(shape)


def _count(shape) -> int:
    return math.prod(shape)


def _layout(shapes):
    """Bytes in all, and for each tensor where its values and scales start
    (values on 16-byte boundaries, scales behind them on the next), its rows
    and its columns."""
    places, at = [], 0
    for shape in shapes:
        c = shape[-1]
        n = math.prod(shape)
        rows = n // c if c else 0
        scales = at + (n + 15) // 16 * 16
        places.append((at, scales, rows, c))
        at = scales + (rows * -(-c // GROUP) + 15) // 16 * 16
    return at, places


def _strides(t: torch.Tensor):
    """(tensor, inner, outer stride, inner stride): row r of the last dimension
    lies at r // inner * outer + r % inner * inner stride."""
    if t.is_contiguous() or t.dim() == 1 and t.stride(0) == 1:
        return t, 1, t.shape[-1], 0
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        t = t.contiguous()
        return t, 1, t.shape[-1], 0
    if t.dim() == 2:
        return t, 1, t.stride(0), 0
    if t.dim() == 3:
        return t, max(t.shape[1], 1), t.stride(0), t.stride(1)
    return t.contiguous(), 1, t.shape[-1], 0


def _check(tensors):
    assert len(tensors) >= 1, "at least one tensor"
    dtype, device = tensors[0].dtype, tensors[0].device
    if dtype not in _TYPES:
        raise TypeError(f"8-bit checkpoints take bf16, fp16 or fp32, got {dtype}")
    for t in tensors:
        if t.dtype != dtype:
            raise TypeError(f"tensors packed together must have one type, got {dtype} and {t.dtype}")
        if not t.is_cuda or t.device != device:
            raise ValueError(f"tensors packed together must be on one CUDA device, got {device} and {t.device}")
        assert t.dim() >= 1, "a tensor needs a last dimension"
    return dtype, device


def _descriptors(rows):
    flat = [v for r in rows for v in r]
    return (ctypes.c_int64 * len(flat))(*flat)


def pack(*tensors: torch.Tensor) -> Packed:
    """The 8-bit form of tensors of one type on one device (up to 4 a launch)."""
    dtype, device = _check(tensors)
    shapes = [tuple(t.shape) for t in tensors]
    total, places = _layout(shapes)
    buffer = torch.empty(total, dtype=torch.uint8, device=device)
    at, rows, keep = buffer.data_ptr(), [], []
    for t, (values, scales, n, c) in zip(tensors, places):
        t, inner, outer_stride, inner_stride = _strides(t.detach())
        keep.append(t)
        rows.append((t.data_ptr(), at + values, at + scales, n, c, inner, outer_stride, inner_stride))
    for i in range(0, len(rows), MAX_TENSORS):
        part = rows[i:i + MAX_TENSORS]
        _call(_native.lib.gdn_checkpoint_pack, device, (_TYPES[dtype], _descriptors(part), len(part)), None)
    return Packed(buffer, dtype, shapes, places)


def unpack_into(packed: Packed, outs: Sequence[torch.Tensor], stream: Optional[int] = None) -> None:
    """Writes the values that `packed` stands for into contiguous tensors of the
    packed shapes and type."""
    assert len(outs) == len(packed)
    device = packed.buffer.device
    at, rows = packed.buffer.data_ptr(), []
    for t, shape, (values, scales, n, c) in zip(outs, packed.shapes, packed.places):
        assert t.shape == shape and t.dtype == packed.dtype and t.is_contiguous()
        if t.device != device:
            raise ValueError(f"an output is on {t.device}, the checkpoint on {device}")
        rows.append((t.data_ptr(), at + values, at + scales, n, c, 1, c, 0))
    for i in range(0, len(rows), MAX_TENSORS):
        part = rows[i:i + MAX_TENSORS]
        _call(_native.lib.gdn_checkpoint_unpack, device, (_TYPES[packed.dtype], _descriptors(part), len(part)),
              stream)


def unpack(packed: Packed) -> List[torch.Tensor]:
    """The tensors that `packed` stands for, in their shapes and type."""
    outs = [torch.empty(s, dtype=packed.dtype, device=packed.buffer.device) for s in packed.shapes]
    unpack_into(packed, outs)
    return outs
