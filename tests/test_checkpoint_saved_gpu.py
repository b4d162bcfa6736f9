"""The 8-bit copies that prefill.run_autograd(checkpoint="int8") keeps are saved
tensors like any others: hooks on saved tensors see them, the backward frees
them although its outputs live on, and a second backward is refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu

T = 4096


def inputs():
    g = torch.Generator().manual_seed(1)
    q, k = (torch.nn.functional.normalize(torch.randn(T, 4, 128, generator=g), dim=-1) for _ in range(2))
    v = torch.randn(T, 8, 128, generator=g)
    a, b = (torch.randn(T, 8, generator=g) for _ in range(2))
    q, k, v, a, b = (t.bfloat16().cuda() for t in (q, k, v, a, b))
    A_log, dt_bias = torch.rand(8, generator=g).cuda(), torch.zeros(8, device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v, A_log, a, dt_bias, b)]
    return leaves, torch.tensor([0, 1000, T], device="cuda")


def forward(gdn, leaves, cu):
    q, k, v, A_log, a, dt_bias, b = leaves
    return gdn.prefill.run_autograd(q, k, v, None, A_log, a, dt_bias, b, cu, None, checkpoint="int8")


PACKED = T * 16 * (128 + 1)     # 16 heads of 128 values and one scale


def test_backward_frees_the_copies(gdn):
    leaves, cu = inputs()
    d_out = torch.ones(T, 8, 128, dtype=torch.bfloat16, device="cuda")
    out, final = forward(gdn, leaves, cu)
    before = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(out, leaves, d_out)
    kept = sum(t.numel() * t.element_size() for t in grads)
    # out, final and their graph are still there
    assert torch.cuda.memory_allocated() <= before + kept - PACKED + 65536
    assert out.grad_fn is not None
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, leaves, d_out)


def test_hooks_see_the_copies(gdn):
    leaves, cu = inputs()
    d_out = torch.ones(T, 8, 128, dtype=torch.bfloat16, device="cuda")
    want = torch.autograd.grad(forward(gdn, leaves, cu)[0], leaves, d_out)
    sizes = []

    def pack(t):
        sizes.append(t.numel() * t.element_size())
        return t.cpu() if t.is_cuda else t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
        out, _ = forward(gdn, leaves, cu)
    assert any(PACKED <= n <= PACKED + 4096 for n in sizes), sizes
    for got, expected in zip(torch.autograd.grad(out, leaves, d_out, retain_graph=True), want):
        assert torch.equal(got, expected)
    # kept for a second backward where that was asked for
    for got, expected in zip(torch.autograd.grad(out, leaves, d_out), want):
        assert torch.equal(got, expected)
