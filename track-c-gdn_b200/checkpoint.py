"""Activation checkpoints in 8 bits.

`pack` turns activations into int8 with one power of two for each 128
neighbouring values of the last dimension (1 + 1/128 bytes a value), `unpack`
turns them back into the type they had.  The scale is the smallest power of
two 2^e with max|v| <= 127 2^e, so a value is off by at most 2^(e-1), less
than max|v| / 126 of its group, and unpacking itself rounds nothing in bf16 and
fp32.  A group that holds a NaN or an infinity unpacks to NaN.

`prefill.run_autograd(..., checkpoint="int8")` and
`recurrence.run_autograd(..., checkpoint="int8")` keep their inputs this way
between forward and backward.  No counterpart in the reference.
"""
from __future__ import annotations

import ctypes
from typing import List, Optional, Sequence

import torch

from . import _native
from .recurrence import _TYPES, _call

GROUP = 128
MAX_TENSORS = 4  # of one launch; more take several


class Packed:
    """Tensors of one type in 8 bits: one buffer, and what was put into it."""

    __slots__ = ("buffer", "dtype", "shapes", "offsets")

    def __init__(self, buffer, dtype, shapes, offsets):
        self.buffer, self.dtype, self.shapes, self.offsets = buffer, dtype, shapes, offsets

    def __len__(self):
        return len(self.shapes)

    def nbytes(self) -> int:
        return self.buffer.numel()

    def values(self, i: int) -> torch.Tensor:
        """The int8 values of tensor i, in its shape (a view of the buffer)."""
        shape, at = self.shapes[i], self.offsets[i]
        return self.buffer[at:at + _count(shape)].view(torch.int8).view(shape)

    def scales(self, i: int) -> torch.Tensor:
        """The exponent bytes E (scale 2^(E-127); 255: not finite) of tensor i,
        [..., ceil(last / 128)] uint8 (a view of the buffer)."""
        shape, at = self.shapes[i], self.offsets[i]
        at += -(-_count(shape) // 16) * 16
        shape = (*shape[:-1], -(-shape[-1] // GROUP))
        return self.buffer[at:at + _count(shape)].view(shape)


def _count(shape) -> int:
    n = 1
    for s in shape:
        n *= s
    return n


def _layout(shapes):
    """Bytes in all, and where each tensor's values and scales start (values on
    16-byte boundaries, scales behind them on the next)."""
    offsets, scales, at = [], [], 0
    for shape in shapes:
        n, c = _count(shape), shape[-1]
        offsets.append(at)
        at += -(-n // 16) * 16
        scales.append(at)
        groups = n // c * -(-c // GROUP) if c else 0
        at += -(-groups // 16) * 16
    return at, offsets, scales


def _strides(t: torch.Tensor):
    """(tensor, inner, outer stride, inner stride): row r of the last dimension
    lies at r // inner * outer + r % inner * inner stride."""
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        t = t.contiguous()
    if t.is_contiguous() or t.dim() == 1:
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


@torch.no_grad()
def pack(*tensors: torch.Tensor) -> Packed:
    """The 8-bit form of tensors of one type on one device (up to 4 a launch)."""
    dtype, device = _check(tensors)
    shapes = [tuple(t.shape) for t in tensors]
    total, offsets, scales = _layout(shapes)
    buffer = torch.empty(total, dtype=torch.uint8, device=device)
    at, rows, keep = buffer.data_ptr(), [], []
    for t, o, s in zip(tensors, offsets, scales):
        t, inner, outer_stride, inner_stride = _strides(t)
        keep.append(t)
        c = t.shape[-1]
        rows.append((t.data_ptr(), at + o, at + s, t.numel() // c if c else 0, c, inner, outer_stride, inner_stride))
    for i in range(0, len(rows), MAX_TENSORS):
        part = rows[i:i + MAX_TENSORS]
        _call("gdn_checkpoint_pack", device, (_TYPES[dtype], _descriptors(part), len(part)), None)
    return Packed(buffer, dtype, shapes, offsets)


def unpack_into(packed: Packed, outs: Sequence[torch.Tensor], stream: Optional[int] = None) -> None:
    """Writes the values that `packed` stands for into contiguous tensors of the
    packed shapes and type."""
    assert len(outs) == len(packed)
    at, rows = packed.buffer.data_ptr(), []
    _, offsets, scales = _layout(packed.shapes)
    for t, shape, o, s in zip(outs, packed.shapes, offsets, scales):
        assert tuple(t.shape) == shape and t.dtype == packed.dtype and t.is_contiguous()
        if t.device != packed.buffer.device:
            raise ValueError(f"an output is on {t.device}, the checkpoint on {packed.buffer.device}")
        c = shape[-1]
        rows.append((t.data_ptr(), at + o, at + s, t.numel() // c if c else 0, c, 1, c, 0))
    for i in range(0, len(rows), MAX_TENSORS):
        part = rows[i:i + MAX_TENSORS]
        _call("gdn_checkpoint_unpack", packed.buffer.device, (_TYPES[packed.dtype], _descriptors(part), len(part)),
              stream)


@torch.no_grad()
def unpack(packed: Packed) -> List[torch.Tensor]:
    """The tensors that `packed` stands for, in their shapes and type."""
    outs = [torch.empty(s, dtype=packed.dtype, device=packed.buffer.device) for s in packed.shapes]
    unpack_into(packed, outs)
    return outs
