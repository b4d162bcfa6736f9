"""8-bit checkpoints of long rows: a flat tensor is one row, of up to 2^31 - 1
values."""
import ctypes

import pytest
import torch


def call(lib, rows, cols):
    arr = (ctypes.c_int64 * 8)(0x100000, 0x10000000000, 0x20000000000, rows, cols, 1, cols, 0)
    got = lib.gdn_checkpoint_pack(0, arr, 1, None)
    assert lib.gdn_checkpoint_unpack(0, arr, 1, None) == got
    return got


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are not real")
def test_sizes(gdn):
    lib = gdn._native.lib
    for rows, cols in ((1, 1 << 24), (1, (1 << 24) + 1), (1, (1 << 31) - 1), (127, (1 << 31) - 1), (7, 1 << 30)):
        assert call(lib, rows, cols) == 6, (rows, cols)           # as far as the missing device
    for rows, cols in ((1, 1 << 31), (1, 1 << 40), (128, (1 << 31) - 1)):
        assert call(lib, rows, cols) == 2, (rows, cols)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [((1 << 24) + 1,), (1 << 25,), (3, (1 << 24) + 130)])
def test_values(gdn, shape):
    """The groups of a long row are those of the same values in short rows, which
    are compared with the definition elsewhere."""
    x = torch.randn(shape, device="cuda").bfloat16()
    for t in (x, x[..., 1:]):              # the second: rows at any address, and, of several, apart
        got, = gdn.checkpoint.unpack(gdn.checkpoint.pack(t))
        assert got.shape == t.shape
        c = t.shape[-1]
        padded = torch.nn.functional.pad(t.reshape(-1, c), (0, -c % 128)).view(-1, 128)
        want, = gdn.checkpoint.unpack(gdn.checkpoint.pack(padded))
        assert torch.equal(got.reshape(-1, c), want.view(-1, c + -c % 128)[:, :c])
