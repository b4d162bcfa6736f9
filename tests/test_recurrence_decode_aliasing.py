"""Outputs of the recurrence's decode that share memory with its inputs or with
one another: refused, but for an output in the very place of an input, whose
elements are read before they are written, and states updated in place."""
import ctypes

import pytest
import torch

import recurrence_ref as ref

P = ctypes.c_void_p
BF16, FP32 = 0, 2
# far apart: x, a, b of a call, its outputs and its states
X, A, B_, OUT, STATE, NEW, INTER = (0x10000000 * n for n in range(1, 8))
PARAMS = P(0x90000000)


def decode(lib, type=BF16, x=X, a=A, b=B_, strides=(64, 64, 64), out=OUT, state=STATE, new=NEW, inter=None, B=4, T=1,
           D=64, slots=None, pool=0):
    p = [None if v is None else P(v) for v in (x, a, b, out, state, new, inter)]
    return lib.gdn_recurrence_decode(type, p[0], strides[0], p[1], strides[1], p[2], strides[2], PARAMS, PARAMS, p[4],
                                     slots, pool, B, T, D, p[3], p[5], p[6], None)


ROW = 64 * 2          # bytes of a row of 64 bf16


def refused(lib):
    """(what, arguments) of calls that answer 7."""
    for T in (1, 4):
        rows = 4 * T
        for at in (X, A, B_):
            yield "out a row later", dict(out=at + ROW, T=T)
            yield "out a row earlier", dict(out=at - ROW, T=T)
            yield "out on the last element", dict(out=at + rows * ROW - 2, T=T)
            yield "new_state on an input", dict(new=at, T=T)
            yield "new_state across an input", dict(new=at + rows * ROW - 4, T=T)
            yield "states after each token on an input", dict(inter=at, T=T)
        yield "out among rows that lie apart", dict(out=X, strides=(192, 64, 64), T=T)
        yield "out in one row that all tokens share", dict(out=X, strides=(0, 64, 64), T=T)
        yield "out on the state", dict(out=STATE + 64, T=T)
        yield "out on the new state", dict(out=NEW, T=T)
        yield "out on the states after each token", dict(out=INTER, inter=INTER, T=T)
    yield "out on a pool", dict(out=STATE + 3 * 256, state=STATE, new=STATE, slots=P(0x91000000), pool=8)


def allowed(lib):
    """Calls that pass the checks."""
    for T in (1, 4):
        for at in (X, A, B_):
            yield "out in the place of an input", dict(out=at, T=T)
        yield "out behind an input", dict(out=X + 4 * T * ROW, T=T)
        yield "out before an input", dict(out=X - 4 * T * ROW, T=T)
        yield "state in place", dict(new=STATE, T=T)
        yield "parts of one projection", dict(x=X, a=X + ROW, b=X + 2 * ROW, strides=(192, 192, 192), T=T)
    yield "out in the place of one row", dict(out=X, B=1, strides=(192, 192, 192), a=X + ROW, b=X + 2 * ROW)


def test_refused(gdn):
    for what, kw in refused(gdn._native.lib):
        assert decode(gdn._native.lib, **kw) == 7, (what, kw)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are not real")
def test_allowed(gdn):
    for what, kw in allowed(gdn._native.lib):
        assert decode(gdn._native.lib, **kw) == 6, (what, kw)     # as far as the missing device


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (3, 1, 130), (300, 1, 128), (5, 4, 36), (40, 7, 256), (3, 64, 33)])
def test_out_in_the_place_of_an_input(gdn, dtype, B, T, D):
    g = torch.Generator().manual_seed(B + T + D)
    x, a, b = (torch.randn(B, T, D, generator=g).to(dtype).cuda() for _ in range(3))
    if T == 1:
        x, a, b = x[:, 0], a[:, 0], b[:, 0]
    A_log, dt_bias = (torch.rand(D, generator=g) * 3 - 5).cuda(), (torch.randn(D, generator=g) * 0.1).cuda()
    state = torch.randn(B, D, generator=g).cuda()
    want, want_new = gdn.recurrence.decode(x, state, A_log, a, dt_bias, b)
    value = ref.forward(*(t.reshape(B * T, D).cpu() if i in (0, 3, 5) else t.cpu()
                          for i, t in enumerate((x, state, A_log, a, dt_bias, b))), list(range(0, B * T + 1, T)))
    ref.assert_close(want, value["out"], "decode", dtype)
    for i in range(3):
        for _ in range(3):
            t = [x.clone(), a.clone(), b.clone()]
            new = torch.empty_like(state)
            gdn.recurrence.decode_into(t[0], state, A_log, t[1], dt_bias, t[2], t[i], new)
            assert torch.equal(t[i], want) and torch.equal(new, want_new)


@pytest.mark.gpu
def test_python_form_refuses(gdn):
    x = torch.randn(9, 64, device="cuda")
    p = torch.zeros(64, device="cuda")
    with pytest.raises(gdn._native.GdnError, match="overlaps"):
        gdn.recurrence.decode_into(x[:8], None, p, x[:8], p, x[:8], x[1:], torch.empty(8, 64, device="cuda"))
