"""Outputs of the recurrence's prefill and backward that share memory with one
another, with the workspace, or with inputs: refused with the aliasing error."""
import ctypes

import pytest
import torch

from test_recurrence_capi import BF16, OK, P, backward, far, prefill

T, D, N = 100, 64, 2                    # the sizes of the calls below
ROWS, STATES = T * D * 2, N * D * 4


def at(n, offset):
    return P(0x10000000 * n + offset)


def test_prefill(gdn):
    lib = gdn._native.lib
    carry, packed = lib.gdn_recurrence_carry_bytes(T, D), lib.gdn_recurrence_packed_bytes(T, D)
    work = lib.gdn_recurrence_workspace_bytes(T, D)
    # out at far(5), final_state at far(9), workspace at far(20)
    for bad in (dict(final=at(5, 0)), dict(final=at(5, ROWS - 4)), dict(final=at(5, 4 - STATES)),
                dict(carries=at(5, ROWS - 16)), dict(carries=at(5, 16 - carry)), dict(packed=at(5, ROWS - 16)),
                dict(packed=at(9, 0)), dict(carries=at(9, STATES - 16)), dict(final=at(20, work - 4)),
                dict(out=at(20, work - 2)), dict(carries=at(20, work - 16)), dict(packed=at(20, 0)),
                dict(carries=far(3), packed=at(3, carry - 16)), dict(packed=far(3), carries=at(3, packed // 16 * 16 - 16)),
                dict(state=at(5, ROWS - 4)), dict(state=at(5, 0))):
        assert prefill(lib, **bad) == 7, bad


def test_backward(gdn):
    lib = gdn._native.lib
    carry = lib.gdn_recurrence_carry_bytes(T, D)
    packed = lib.gdn_recurrence_packed_bytes(T, D)
    work = lib.gdn_recurrence_backward_workspace_bytes(T, D)
    # dx, da, db at far(5) to far(7), workspace at far(20)
    for bad in (dict(da=far(5)), dict(db=far(5)), dict(db=far(6)), dict(da=at(5, ROWS - 2)), dict(db=at(6, 2 - ROWS)),
                dict(d_state=at(5, ROWS - 4)), dict(d_state=at(7, 0)), dict(state=at(6, 0)), dict(d_final=at(6, 4)),
                dict(state=at(20, work - 4)), dict(dx=at(20, work - 2)), dict(d_state=at(20, 0)),
                dict(carries=at(5, 0)), dict(carries=at(20, work // 16 * 16 - 16)),
                dict(packed=at(7, ROWS - 16), carries=far(3)), dict(packed=far(3), carries=at(20, 0)),
                dict(packed=far(3), carries=far(4), dx=at(3, packed - 1 & ~1)), dict(carries=far(3), db=at(3, carry - 2))):
        assert backward(lib, **bad) == 7, bad


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are not real")
def test_side_by_side(gdn):
    """One next to the other is as good as far apart."""
    lib = gdn._native.lib
    carry = lib.gdn_recurrence_carry_bytes(T, D)
    work = lib.gdn_recurrence_workspace_bytes(T, D)
    bwork = lib.gdn_recurrence_backward_workspace_bytes(T, D)
    for good in (dict(final=at(5, ROWS)), dict(final=at(5, -STATES)), dict(carries=at(5, ROWS)),
                 dict(packed=far(3), carries=at(3, -carry)), dict(final=at(20, work)), dict(state=far(9)),
                 dict(state=at(5, ROWS))):
        assert prefill(lib, **good) == 6, good
    for good in (dict(da=at(5, ROWS), db=at(5, 2 * ROWS)), dict(d_state=at(7, ROWS)), dict(state=at(5, -STATES)),
                 dict(d_state=at(20, bwork)), dict(carries=at(5, ROWS))):
        assert backward(lib, **good) == 6, good


@pytest.mark.gpu
def test_python_forms(gdn):
    rec = gdn.recurrence
    x = torch.randn(700, 64, device="cuda")
    p = torch.zeros(64, device="cuda")
    out = torch.empty_like(x)
    ws, bws = rec.alloc_workspace(700, 64, "cuda"), rec.alloc_backward_workspace(700, 64, "cuda")
    with pytest.raises(gdn._native.GdnError, match="overlaps"):
        rec.run_into(x, None, p, x, p, x, None, out, out[699:], ws)
    g = [torch.empty_like(x) for _ in range(2)] + [torch.empty_like(p) for _ in range(2)]
    with pytest.raises(gdn._native.GdnError, match="overlaps"):
        rec.backward_into(x, None, p, x, p, x, None, x, None, g[0], g[1], g[0], g[2], g[3], None, bws)
