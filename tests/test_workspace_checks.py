"""What the Python forms hand to the C ABI for a caller's workspace: an address
on a 1024-byte boundary and the bytes that are left from there on, which a
buffer shorter than its alignment slack does not have."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p
OK = P(0x100000)


def at(offset, size, dtype=torch.uint8):
    """A tensor of `size` elements that starts `offset` bytes behind a 1024-byte boundary."""
    buf = torch.empty(4096, dtype=torch.uint8)
    start = -buf.data_ptr() % 1024 + offset
    return buf[start:start + size * dtype.itemsize].view(dtype)


@pytest.mark.parametrize("offset", [0, 64, 512, 960])
@pytest.mark.parametrize("size", [0, 16, 100, 512, 1500])
def test_bytes_behind_the_boundary(gdn, offset, size):
    ws = at(offset, size)
    ptr, left = gdn._native.aligned_workspace(ws, ws.device)
    assert ptr % 1024 == 0
    assert left == max(0, size - -offset % 1024)


def test_bytes_of_other_types(gdn):
    ws = at(512, 300, torch.float32)
    assert gdn._native.aligned_workspace(ws, ws.device)[1] == 1200 - 512


def test_short_workspace_is_refused(gdn):
    """Each entry point answers that the workspace is too small (4), before it
    looks for a device."""
    lib = gdn._native.lib
    ws = gdn._native.aligned_workspace(at(512, 100), torch.device("cpu"))
    far = [P(0x10000000 * n) for n in range(1, 9)]
    assert lib.gdn_recurrence_prefill(0, OK, 64, OK, 64, OK, 64, OK, OK, None, None, 0, OK, 2, 100, 64, 0, far[0],
                                      far[1], None, None, *ws, None) == 4
    assert lib.gdn_recurrence_backward(0, OK, 64, OK, 64, OK, 64, None, OK, OK, None, OK, 2, 100, 64, 0, OK, 64, None,
                                       None, *far[:3], OK, OK, None, *ws, None) == 4
    assert lib.gdn_prefill_qk4_v8_d128_k_last(OK, OK, OK, None, OK, OK, OK, OK, OK, 2, 128, 0.0, OK, OK, *ws,
                                              None) == 4
    assert lib.gdn_prefill_pool_qk4_v8_d128_k_last(OK, OK, OK, OK, 8, OK, OK, OK, OK, OK, OK, 2, 128, 0.0, OK, *ws,
                                                   None) == 4
    assert lib.gdn_prefill_backward_qk4_v8_d128_k_last(OK, OK, OK, None, OK, OK, OK, OK, OK, 2, 128, 0.0, OK, None,
                                                       *[OK] * 7, None, *ws, None) == 4


def test_other_device_and_gaps_are_refused(gdn):
    ws = torch.empty(4096, dtype=torch.uint8)
    with pytest.raises(ValueError, match="workspace"):
        gdn._native.aligned_workspace(ws, torch.device("cuda", 0))
    with pytest.raises(AssertionError, match="contiguous"):
        gdn._native.aligned_workspace(ws[::2], ws.device)


@pytest.mark.gpu
def test_calls_refuse_such_workspaces(gdn):
    import cases
    from gpu_util import prefill_args

    rec, pre = gdn.recurrence, gdn.prefill
    x = torch.randn(700, 64, device="cuda")
    p = torch.zeros(64, device="cuda")
    out, final = torch.empty_like(x), torch.empty(1, 64, device="cuda")
    g = [torch.empty_like(x) for _ in range(3)] + [torch.empty_like(p) for _ in range(2)] + [None]
    q = prefill_args(cases.prefill_inputs(seed=3, lens=[100, 30], with_state=True))
    p_out, p_final = torch.empty(130, 8, 128, dtype=torch.bfloat16, device="cuda"), torch.empty_like(q[3])
    d_out = torch.zeros_like(p_out)
    dev = torch.empty(1, device="cuda").device
    f32 = [torch.empty(s, device="cuda") for s in ((130, 4, 128), (130, 4, 128), (130, 8, 128), (130, 8), (130, 8),
                                                   (8,), (8,))]
    slots = torch.arange(2, dtype=torch.int32, device="cuda")
    calls = [
        (lambda ws: rec.run_into(x, None, p, x, p, x, None, out, final, ws), rec.alloc_workspace(700, 64, dev)),
        (lambda ws: rec.run_pool_into(x, final, slots[:1], p, x, p, x, None, out, ws),
         rec.alloc_workspace(700, 64, dev)),
        (lambda ws: rec.backward_into(x, None, p, x, p, x, None, x, None, *g, ws),
         rec.alloc_backward_workspace(700, 64, dev)),
        (lambda ws: pre.prefill_into(*q, None, p_out, p_final, ws), pre.alloc_workspace(130, 2, dev)),
        (lambda ws: pre.prefill_pool_into(*q[:3], p_final, slots, *q[4:], None, p_out, ws),
         pre.alloc_workspace(130, 2, dev)),
        (lambda ws: pre.backward_into(*q, None, d_out, None, *f32, None, ws),
         pre.alloc_backward_workspace(130, 2, dev)),
    ]
    for call, ws in calls:
        base = -ws.data_ptr() % 1024
        for short in (ws[:0], ws[base:base + 512], ws[base + 512:base + 612], ws[base + 8:base + 1032]):
            with pytest.raises(gdn._native.GdnError, match="workspace|NULL"):     # an empty tensor has no address
                call(short)
        with pytest.raises(ValueError, match="workspace"):
            call(ws.cpu())
        call(ws)
    torch.cuda.synchronize()
    assert gdn._native.read_device_status() == 0
