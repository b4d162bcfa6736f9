"""The recurrence's and the checkpoints' C entry points and Python checks where
no GPU is needed: sizes, NULL pointers, alignment, workspaces, aliasing; and
the float64 reference of the GPU tests against torch's own differentiation."""
import ctypes

import pytest
import torch

import recurrence_ref as ref

P = ctypes.c_void_p
OK = P(0x100000)
BF16, FP32 = 0, 2
BIG = 1 << 40


def far(n):
    return P(0x10000000 * n)


def prefill(lib, type=BF16, x=OK, xs=64, a=OK, b=OK, A_log=OK, dt_bias=OK, state=None, slots=None, pool=0, cu=OK,
            N=2, T=100, D=64, out=far(5), final=far(9), carries=None, packed=None, ws=far(20), ws_bytes=BIG):
    return lib.gdn_recurrence_prefill(type, x, xs, a, 64, b, 64, A_log, dt_bias, state, slots, pool, cu, N, T, D, 0,
                                      out, final, carries, packed, ws, ws_bytes, None)


def test_prefill_arguments(gdn):
    lib = gdn._native.lib
    for bad in (dict(type=3), dict(type=-1), dict(T=-1), dict(N=-1), dict(D=0), dict(D=-4), dict(T=(1 << 31) + 1),
                dict(N=0), dict(cu=None, N=3), dict(slots=OK, pool=0, state=far(9)), dict(T=1 << 31, D=1 << 24)):
        assert prefill(lib, **bad) == 2, bad
    assert prefill(lib, N=0, T=0) == 0
    for bad in (dict(x=None), dict(a=None), dict(b=None), dict(A_log=None), dict(dt_bias=None), dict(out=None),
                dict(final=None), dict(ws=None), dict(slots=OK, pool=4)):
        assert prefill(lib, **bad) == 1, bad
    for bad in (dict(x=P(0x100001)), dict(type=FP32, x=P(0x100002)), dict(A_log=P(0x100002)), dict(cu=P(0x100004)),
                dict(final=P(0x90000002)), dict(carries=P(0x100008)), dict(packed=P(0x100004)), dict(state=P(0x100001))):
        assert prefill(lib, **bad) == 3, bad
    assert prefill(lib, ws=P(0x10000200)) == 4
    need = lib.gdn_recurrence_workspace_bytes(100, 64)
    assert need > 0 and prefill(lib, ws_bytes=need - 1) == 4
    assert prefill(lib, state=P(0x90000000 - 256)) == 7
    for out in (OK, P(0x100000 + 99 * 128), P(0x100000 - 64)):
        assert prefill(lib, out=out) == 7


def test_negative_strides(gdn):
    lib = gdn._native.lib
    assert prefill(lib, xs=-64) == 2
    for i in (2, 4, 6):
        args = [BF16, OK, 64, OK, 64, OK, 64, OK, OK]
        args[i] = -1
        assert lib.gdn_recurrence_prefill(*args, None, None, 0, OK, 2, 100, 64, 0, far(5), far(9), None, None, far(20),
                                          BIG, None) == 2
        assert lib.gdn_recurrence_decode(*args, None, None, 0, 4, 1, 64, OK, far(3), None, None) == 2
        args[7:7] = [None]
        assert lib.gdn_recurrence_backward(*args, None, OK, 2, 100, 64, 0, OK, 64, None, None, far(5), far(6), far(7),
                                           OK, OK, None, far(20), BIG, None) == 2
    assert lib.gdn_recurrence_backward(BF16, OK, 64, OK, 64, OK, 64, None, OK, OK, None, OK, 2, 100, 64, 0, OK, -64,
                                       None, None, far(5), far(6), far(7), OK, OK, None, far(20), BIG, None) == 2


def backward(lib, type=BF16, x=OK, a=OK, b=OK, packed=None, state=None, cu=OK, N=2, T=100, D=64, d_out=OK,
             d_final=None, carries=None, dx=far(5), da=far(6), db=far(7), dA=OK, ddt=OK, d_state=None, ws=far(20), ws_bytes=BIG):
    return lib.gdn_recurrence_backward(type, x, 64, a, 64, b, 64, packed, OK, OK, state, cu, N, T, D, 0, d_out, 64,
                                       d_final, carries, dx, da, db, dA, ddt, d_state, ws, ws_bytes, None)


def test_backward_arguments(gdn):
    lib = gdn._native.lib
    for bad in (dict(type=7), dict(T=-1), dict(D=0), dict(N=0), dict(cu=None, N=3)):
        assert backward(lib, **bad) == 2, bad
    for bad in (dict(x=None), dict(d_out=None), dict(dx=None), dict(db=None), dict(dA=None), dict(ddt=None),
                dict(ws=None), dict(packed=OK)):            # 8 bits need the forward's states
        assert backward(lib, **bad) == 1, bad
    for bad in (dict(d_out=P(0x100001)), dict(dA=P(0x100002)), dict(d_state=P(0x100002)), dict(carries=P(0x100004))):
        assert backward(lib, **bad) == 3, bad
    need = lib.gdn_recurrence_backward_workspace_bytes(100, 64)
    assert need > lib.gdn_recurrence_workspace_bytes(100, 64)
    assert backward(lib, ws_bytes=need - 1) == 4 and backward(lib, ws=P(0x10000010)) == 4
    assert backward(lib, state=far(3), d_state=P(0x30000000 + 16)) == 7
    assert backward(lib, d_final=far(3), d_state=P(0x30000000 + 16)) == 7
    assert backward(lib, d_final=far(3), d_state=far(3)) == 7
    assert backward(lib, dx=OK) == 7 and backward(lib, db=P(0x100000 + 99 * 128)) == 7


def decode(lib, type=BF16, x=OK, state=None, slots=None, pool=0, B=4, T=1, D=64, out=OK, new=far(3), inter=None):
    return lib.gdn_recurrence_decode(type, x, 64, OK, 64, OK, 64, OK, OK, state, slots, pool, B, T, D, out, new, inter,
                                     None)


def test_decode_arguments(gdn):
    lib = gdn._native.lib
    for bad in (dict(type=5), dict(B=-1), dict(T=0), dict(T=65), dict(D=0), dict(slots=OK, state=far(3)),
                dict(B=1 << 24, D=1 << 24)):
        assert decode(lib, **bad) == 2, bad
    assert decode(lib, B=0) == 0
    for bad in (dict(x=None), dict(out=None), dict(new=None), dict(slots=OK, pool=5)):
        assert decode(lib, **bad) == 1, bad
    assert decode(lib, new=P(0x30000002)) == 3
    assert decode(lib, state=P(0x30000010)) == 7
    assert decode(lib, inter=P(0x30000010)) == 7


def tensor(data=0x100000, values=0x200000, scales=0x300000, rows=4, cols=128, inner=1):
    return [data, values, scales, rows, cols, inner, 128, 0]


def test_checkpoint_arguments(gdn):
    lib = gdn._native.lib

    def call(*tensors, type=BF16, count=None):
        flat = [v for t in tensors for v in t]
        arr = (ctypes.c_int64 * len(flat))(*flat) if flat else None
        n = len(tensors) if count is None else count
        got = lib.gdn_checkpoint_pack(type, arr, n, None)
        assert lib.gdn_checkpoint_unpack(type, arr, n, None) == got
        return got

    assert call() == 0 and call(tensor(rows=0)) == 0 and call(tensor(cols=0)) == 0
    assert call(tensor(), type=9) == 2 and call(*[tensor()] * 5) == 2 and call(count=-1) == 2
    assert call(tensor(rows=-1)) == 2 and call(tensor(inner=0)) == 2 and call(tensor(rows=1 << 39)) == 2
    assert call(count=1) == 1
    assert call(tensor(data=0)) == 1 and call(tensor(values=0)) == 1 and call(tensor(scales=0)) == 1
    assert call(tensor(data=0x100001)) == 3


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-device path")
def test_no_device_is_reported(gdn):
    assert prefill(gdn._native.lib) == 6
    assert backward(gdn._native.lib) == 6
    assert decode(gdn._native.lib) == 6


def test_python_checks(gdn):
    rec, ck = gdn.recurrence, gdn.checkpoint
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    p = torch.zeros(8)
    with pytest.raises(TypeError, match="x"):
        rec.run(x.long(), None, p, x, p, x)
    with pytest.raises(TypeError, match="type"):
        rec.run(x, None, p, x.float(), p, x)
    with pytest.raises(TypeError, match="fp32"):
        rec.run(x, None, p.double(), x, p, x)
    with pytest.raises(ValueError, match="CUDA"):
        rec.run(x, None, p, x, p, x)
    with pytest.raises(ValueError, match="int8"):
        rec.run_autograd(x, None, p, x, p, x, checkpoint="fp4")
    with pytest.raises(ValueError, match="int8"):
        gdn.prefill.run_autograd(*[None] * 10, checkpoint="fp4")
    with pytest.raises(ValueError, match="CUDA"):
        ck.pack(x)
    with pytest.raises(TypeError):
        ck.pack(x.long())
    with pytest.raises(AssertionError):
        ck.pack()
    with pytest.raises(AssertionError, match="packed"):
        rec._sequences(x.view(2, 2, 8), torch.zeros(3, dtype=torch.int64))


@pytest.mark.parametrize("eight", [False, True])
def test_reference_gradients_against_autograd_and_differences(eight):
    """The formulas of recurrence_ref.backward against torch.autograd of the
    recurrence (of its restarted form with 8-bit values), and that against
    differences."""
    lens, D = [70, 0, 3, 64], 5
    cu = [0, 70, 70, 73, 137]
    g = torch.Generator().manual_seed(1)
    x, a, b = (torch.randn(137, D, generator=g) for _ in range(3))
    A_log, dt_bias = torch.randn(D, generator=g), torch.randn(D, generator=g) * 0.1
    state = torch.randn(4, D, generator=g)
    d_out, d_final = torch.randn(137, D, generator=g), torch.randn(4, D, generator=g)
    want = ref.backward(x, state, A_log, a, dt_bias, b, cu, d_out, d_final, eight)
    exact = ref.forward(x, state, A_log, a, dt_bias, b, cu)["out"][0]
    q = ref.quantise if eight else lambda t: t.double()
    leaves = [t.double().requires_grad_(True) for t in (q(x), state, A_log, q(a), dt_bias, q(b))]

    def loss(x, state, A_log, a, dt_bias, b):
        total = 0.0
        for n, (s, e) in enumerate(ref.ranges(cu)):
            h = state[n]
            for t in range(s, e):
                if eight and t > s and t % ref.CHUNK == 0:
                    h = h + (exact[t - 1] - h).detach()      # restarted: its value, not its gradient
                h = torch.exp(-A_log.exp() * ref.softplus(a[t] + dt_bias)) * h + torch.sigmoid(b[t]) * x[t]
                total = total + (h * d_out[t]).sum()
            total = total + (h * d_final[n]).sum()
        return total

    grads = torch.autograd.grad(loss(*leaves), leaves)
    for name, got in zip(("dx", "d_state", "dA_log", "da", "ddt_bias", "db"), grads):
        torch.testing.assert_close(want[name][0], got, rtol=1e-9, atol=1e-12)
    if not eight:
        v = [torch.randn(t.shape, generator=g).double() for t in leaves]
        e = 1e-5
        diff = (loss(*(t + e * d for t, d in zip(leaves, v))) - loss(*(t - e * d for t, d in zip(leaves, v)))) / (2 * e)
        along = sum((p * d).sum() for p, d in zip(grads, v))
        # e^2 of third derivatives, and 1e-16 / e of rounding
        assert abs(diff - along) < 1e-6 * sum((p * d).abs().sum() for p, d in zip(grads, v))
