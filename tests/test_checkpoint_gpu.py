"""Activation checkpoints in 8 bits on the GPU: the format is exact arithmetic,
so values and scales have to be those of the definition, bit for bit."""
import pytest
import torch

import recurrence_ref as ref

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def same(got, want):
    want = want.to(got.dtype)
    return bool(((got.cpu() == want) | (got.cpu().isnan() & want.isnan())).all())


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", [(1,), (128,), (3, 1), (1, 128), (7, 129), (5, 4, 128), (33, 64), (2, 3, 260),
                                   (4, 3, 2, 100), (1000, 8, 128)])
def test_round_trip(gdn, dtype, shape):
    g = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(shape, generator=g) * torch.exp(1.5 * torch.randn(*shape[:-1], 1, generator=g))).to(dtype)
    packed = gdn.checkpoint.pack(x.cuda())
    got, = gdn.checkpoint.unpack(packed)
    assert got.shape == x.shape and got.dtype == dtype
    assert same(got, ref.quantise(x))
    assert packed.values(0).shape == x.shape and packed.values(0).dtype == torch.int8
    E = packed.scales(0).cpu().int()
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), (E - 127).double())
    unit = unit.repeat_interleave(128, -1)[..., :shape[-1]]
    assert bool((packed.values(0).cpu().double() * unit == ref.quantise(x)).all())
    # half a unit, less than max|x| / 126 of the group
    assert bool(((got.cpu().double() - x.double()).abs() <= unit / 2).all())


def test_special_values(gdn):
    """Zeros, the largest and smallest numbers, ties, and groups that are not
    finite beside groups that are."""
    for dtype in (BF16, FP16, FP32):
        top, low = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
        rows = torch.zeros(12, 256, dtype=dtype)
        rows[1, 3] = top
        rows[2, :5] = torch.tensor([top, -top, top / 2, 1.0, low], dtype=dtype)
        rows[3, 7] = low
        rows[4, :128] = torch.arange(128).to(dtype) / 64
        rows[5, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5]).to(dtype)      # unit 1: ties to even
        rows[6, :3] = torch.tensor([127.5, 63.0, -127.5]).to(dtype)
        rows[7, 0], rows[7, 200] = float("nan"), 2.0
        rows[8, 130], rows[8, 5] = float("inf"), -3.0
        rows[9, 0] = -float("inf")
        rows[10, :2] = torch.tensor([2.0 ** -24, 2.0 ** -23]).to(dtype)
        rows[11, :] = -0.0
        got, = gdn.checkpoint.unpack(gdn.checkpoint.pack(rows.cuda()))
        assert same(got, ref.quantise(rows)), dtype
        assert torch.isfinite(got[:7]).all()
        assert got[7, :128].isnan().all() and got[7, 200] == 2.0
        assert got[8, 128:].isnan().all() and got[8, 5] == -3.0


def test_strided_inputs_and_many_tensors(gdn):
    g = torch.Generator().manual_seed(3)
    joint = torch.randn(50, 2048, generator=g).to(BF16).cuda()
    q, k, v = (t.unflatten(1, (-1, 128)) for t in joint.split([512, 512, 1024], 1))
    odd = torch.randn(9, 77, generator=g).to(BF16).cuda()[:, 3:]
    turned = torch.randn(64, 30, generator=g).to(BF16).cuda().t()
    empty = torch.empty(0, 128, dtype=BF16, device="cuda")
    none = torch.empty(3, 0, dtype=BF16, device="cuda")
    tensors = (q, k, v, odd, turned, empty, none)
    packed = gdn.checkpoint.pack(*tensors)
    assert len(packed) == 7 and packed.nbytes() < sum(t.numel() for t in tensors) * 1.05 + 500
    for t, got in zip(tensors, gdn.checkpoint.unpack(packed)):
        assert got.shape == t.shape and got.is_contiguous()
        if t.numel():
            assert same(got, ref.quantise(t.cpu()))


def test_checkpointed_prefill_gradients(gdn):
    """GDN prefill with 8-bit checkpoints: the same outputs, and exactly the
    gradients of the backward at the restored q, k and v."""
    import cases
    from gpu_util import prefill_args

    args = prefill_args(cases.prefill_inputs(seed=5, lens=[90, 0, 140], with_state=True))
    q, k, v, state, A_log, a, dt, b, cu = args
    g = torch.Generator().manual_seed(1)
    d_out = (torch.randn(230, 8, 128, generator=g) * 0.1).to(BF16).cuda()
    d_final = (torch.randn(3, 8, 128, 128, generator=g) * 0.01).cuda()
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, state, A_log, a, dt, b)]
    out, final = gdn.prefill.run_autograd(*leaves, cu, None, checkpoint="int8")
    ref_out, ref_final = gdn.prefill.run(*args, None)
    assert torch.equal(out, ref_out) and torch.equal(final, ref_final)
    grads = torch.autograd.grad((out, final), leaves, (d_out, d_final))
    q8, k8, v8 = (ref.quantise(t.cpu()).to(BF16).cuda() for t in (q, k, v))
    want = gdn.prefill.backward(q8, k8, v8, state, A_log, a, dt, b, cu, None, d_out, d_final)
    for got, leaf, name in zip(grads, leaves, ("dq", "dk", "dv", "d_state", "dA_log", "da", "ddt_bias", "db")):
        assert got.dtype == leaf.dtype and torch.equal(got, want[name].to(leaf.dtype).view_as(leaf)), name


def test_two_streams_and_capture(gdn):
    x = torch.randn(3000, 1024, device="cuda").to(BF16)
    want, = gdn.checkpoint.unpack(gdn.checkpoint.pack(x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, = gdn.checkpoint.unpack(gdn.checkpoint.pack(x))
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = gdn.checkpoint.unpack(gdn.checkpoint.pack(x))
    x.mul_(0.37)
    graph.replay()
    torch.cuda.synchronize()
    want, = gdn.checkpoint.unpack(gdn.checkpoint.pack(x))
    assert torch.equal(got, want)
