"""Calls from a thread whose current CUDA context is one of the caller's own
(cuCtxCreate), as a program on the driver interface has: they run there, where
the caller's memory and streams are valid, and leave it current.

Each part runs in a process of its own.  The first call touches nothing but
portable pinned memory, which is valid in any context; kernels follow only when
the context has been seen to stay."""
import ctypes
import importlib
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent
P = ctypes.c_void_p


class Driver:
    """A context on device 0, current from its creation on, and memory in it."""

    def __init__(self):
        self.cu = ctypes.CDLL("libcuda.so.1")
        self.ok("cuInit", 0)
        dev = ctypes.c_int()
        self.ok("cuDeviceGet", ctypes.byref(dev), 0)
        self.ctx = P()
        self.ok("cuCtxCreate_v2", ctypes.byref(self.ctx), 0, dev)

    def ok(self, name, *args):
        status = getattr(self.cu, name)(*args)
        assert status == 0, f"{name}: {status}"

    def current(self):
        ctx = P()
        self.ok("cuCtxGetCurrent", ctypes.byref(ctx))
        return ctx.value

    def alloc(self, nbytes):
        p = ctypes.c_uint64()
        self.ok("cuMemAlloc_v2", ctypes.byref(p), ctypes.c_size_t(nbytes))
        return P(p.value)

    def put(self, array):
        p = self.alloc(array.nbytes)
        self.ok("cuMemcpyHtoD_v2", p, array.ctypes.data_as(P), ctypes.c_size_t(array.nbytes))
        return p

    def get(self, p, like):
        import numpy as np
        got = np.empty_like(like)
        self.ok("cuCtxSynchronize")
        self.ok("cuMemcpyDtoH_v2", got.ctypes.data_as(P), p, ctypes.c_size_t(got.nbytes))
        return got

    def pinned(self, nbytes):
        p = P()
        portable_and_mapped = 1 | 2
        self.ok("cuMemHostAlloc", ctypes.byref(p), ctypes.c_size_t(nbytes), portable_and_mapped)
        return p


def start(gdn):
    """A context in which a first call has been seen to stay."""
    d = Driver()
    assert d.current() == d.ctx.value
    p = d.pinned(4096)
    ok = P(0x100000)
    # no sequences: two memsets of the parameters' gradients and nothing else
    st = gdn._native.lib.gdn_recurrence_backward(
        2, None, 8, None, 8, None, 8, None, ok, ok, None, None, 0, 0, 8, 0, None, 8, None, None, None, None, None,
        p, P(p.value + 64), None, P(0x10000000), 1 << 40, None)
    assert st == 0
    assert d.current() == d.ctx.value, "the call replaced the caller's context"
    d.ok("cuCtxSynchronize")
    return d


def rows(T, D, seed):
    import numpy as np
    rng = np.random.default_rng(seed)
    x, a, b = (rng.standard_normal((T, D)).astype(np.float32) for _ in range(3))
    return x, a, b, rng.standard_normal(D).astype(np.float32) - 2, rng.standard_normal(D).astype(np.float32)


def decode_in_own_context(gdn):
    import numpy as np
    B, D = 5, 40
    x, a, b, A_log, dt_bias = rows(B, D, 1)
    d = start(gdn)
    dx, da, db, dA, ddt = (d.put(t) for t in (x, a, b, A_log, dt_bias))
    out, new = d.put(np.full_like(x, 7)), d.put(np.full_like(x, 7))
    st = gdn._native.lib.gdn_recurrence_decode(2, dx, D, da, D, db, D, dA, ddt, None, None, 0, B, 1, D, out, new, None,
                                               None)
    assert st == 0
    want = x.astype(np.float64) / (1 + np.exp(-b.astype(np.float64)))
    # one product of a sigmoid with relative error (2 |b| + 8) 2^-24, |b| < 5
    assert (np.abs(d.get(out, x) - want) <= np.abs(want) * 20 * 2.0 ** -24 + 1e-30).all()
    assert np.array_equal(d.get(new, x), d.get(out, x))
    assert d.current() == d.ctx.value


def recurrence_after_the_primary_context(gdn):
    """Forward and backward first through torch, then in a context of the
    caller's own, then in another: kernels with much shared memory have to be
    allowed it in each."""
    import numpy as np
    import torch

    T, D = 1000, 64
    host = rows(T, D, 2)
    x, a, b, A_log, dt_bias = (torch.from_numpy(t).cuda() for t in host)
    want, want_final = gdn.recurrence.run(x, None, A_log, a, dt_bias, b)
    grads = gdn.recurrence.backward(x, None, A_log, a, dt_bias, b, None, x)
    want, want_final = want.cpu().numpy(), want_final.cpu().numpy()
    grads = {k: v.cpu().numpy() for k, v in grads.items() if v is not None}
    lib = gdn._native.lib
    need, bneed = lib.gdn_recurrence_workspace_bytes(T, D), lib.gdn_recurrence_backward_workspace_bytes(T, D)
    for _ in range(2):
        d = start(gdn)
        dx, da, db, dA, ddt = (d.put(t) for t in host)
        out, final = d.alloc(want.nbytes), d.alloc(want_final.nbytes)
        ws, bws = (P(-(-d.alloc(n + 1024).value // 1024) * 1024) for n in (need, bneed))
        assert lib.gdn_recurrence_prefill(2, dx, D, da, D, db, D, dA, ddt, None, None, 0, None, 1, T, D, 0, out, final,
                                          None, None, ws, need, None) == 0
        assert np.array_equal(d.get(out, want), want) and np.array_equal(d.get(final, want_final), want_final)
        g = {k: d.alloc(v.nbytes) for k, v in grads.items()}
        assert lib.gdn_recurrence_backward(2, dx, D, da, D, db, D, None, dA, ddt, None, None, 1, T, D, 0, dx, D, None,
                                           None, g["dx"], g["da"], g["db"], g["dA_log"], g["ddt_bias"], g["d_state"], bws,
                                           bneed, None) == 0
        for k, v in grads.items():
            assert np.array_equal(d.get(g[k], v), v), k
        assert d.current() == d.ctx.value
        d.ok("cuCtxDestroy_v2", d.ctx)
    # torch's context is the one below: back to it
    again, _ = gdn.recurrence.run(x, None, A_log, a, dt_bias, b)
    assert np.array_equal(again.cpu().numpy(), want)


def run_part(name):
    res = subprocess.run([sys.executable, __file__, name], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-3000:]
    assert "part ok" in res.stdout


def test_first_call_leaves_the_context_current():
    run_part("start")


def test_decode_in_own_context():
    run_part("decode_in_own_context")


def test_recurrence_after_the_primary_context():
    run_part("recurrence_after_the_primary_context")


if __name__ == "__main__":
    sys.path.insert(0, str(ROOT))
    package = importlib.import_module("track-c-gdn_b200")
    globals()[sys.argv[1]](package)
    print("part ok")
