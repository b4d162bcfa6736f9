"""The channelwise recurrence against its definition in each way that a call can
take through the kernels: one launch or chunks joined through the workspace, by
groups of one or of eight; rows fetched by tensor copies, row by row, or directly;
with and without 8-bit copies.  Where the way depends on sizes, the test reads
back from the workspace's header that it was the one meant.

Bounds are those of recurrence_ref.py: they count roundings, and hold for any
order in which affine maps are composed."""
import pytest
import torch

import recurrence_ref as ref
from test_recurrence_gpu import check_forward, check_gradients, cumulative, dev, inputs

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ("dx", "d_state", "dA_log", "da", "ddt_bias", "db")
EMPTY = 0x5a5a5a5a          # what a workspace holds that no call has written to


@pytest.fixture(autouse=True)
def _clean_status(gdn):
    gdn._native.read_device_status()
    yield
    assert gdn._native.read_device_status() == 0


def header(ws):
    """(streams, chunks to a published state) that the call's first launch chose;
    None if there was none."""
    at = -ws.data_ptr() % 1024
    bad, streams, group = ws[at:at + 12].cpu().clone().view(torch.int32).tolist()
    assert bad in (0, EMPTY)
    return None if streams == EMPTY else (streams, group)


def forward(gdn, args, cu, packed=None):
    """run_into, with 8-bit copies too; returns (out, final_state) and the header."""
    x = args[0]
    ws = gdn.recurrence.alloc_workspace(*x.shape, "cuda")
    ws.fill_(0x5a)
    out, final = torch.empty(x.shape, dtype=x.dtype, device="cuda"), torch.empty(len(cu) - 1, x.shape[1], device="cuda")
    gdn.recurrence._prefill(*args, cu.cuda(), out, final, ws, packed=packed)
    return (out, final), header(ws)


def backward(gdn, args, cu, d_out, d_final):
    x = args[0]
    ws = gdn.recurrence.alloc_backward_workspace(*x.shape, "cuda")
    ws.fill_(0x5a)
    rows = [torch.empty(x.shape, dtype=x.dtype, device="cuda") for _ in range(3)]
    sums = [torch.empty(x.shape[1], device="cuda") for _ in range(2)]
    d_state = torch.empty(len(cu) - 1, x.shape[1], device="cuda")
    gdn.recurrence.backward_into(*args, cu.cuda(), d_out, d_final, *rows, *sums, d_state, ws)
    return dict(zip(("dx", "da", "db", "dA_log", "ddt_bias", "d_state"), (*rows, *sums, d_state))), header(ws)


def grads_of(lens, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(sum(lens), D, generator=g).to(dtype), torch.randn(len(lens), D, generator=g)


# ---------------------------------------------------------------------------
# the limit of the one launch
# ---------------------------------------------------------------------------
LIMITS = [      # type, channels, 8-bit copies, chunks of one sequence, of several
    (BF16, 128, False, 8, 7),
    (FP16, 136, False, 8, 7),
    (FP32, 128, False, 5, 4),
    (BF16, 132, False, 5, 5),
    (FP32, 130, False, 3, 3),
    (BF16, 128, True, 3, 3),
    (FP32, 128, True, 2, 2),
    (FP16, 132, True, 2, 2),
    (FP32, 130, True, 1, 1),
]


@pytest.mark.parametrize("dtype,D,eight,one,several", LIMITS)
@pytest.mark.parametrize("sequences", [1, 3, 1024, 1025])
def test_one_launch_for_short_inputs(gdn, dtype, D, eight, one, several, sequences):
    limit = 64 * (one if sequences == 1 else several)
    for T in (limit, limit + 1):
        lens = [T] if sequences == 1 else [0] * (sequences - 3) + [T // 3, 0, T - T // 3]
        args = inputs(lens, D, dtype, T, slow=True)
        cu = cumulative(lens)
        packed = None
        if eight:
            packed = torch.empty(gdn.recurrence._saved_bytes(T, D)[1], dtype=torch.uint8, device="cuda")
        got, head = forward(gdn, dev(args), cu, packed)
        assert (head is None) == (T == limit and sequences <= 1024), (T, head)
        check_forward(got, args, cu, f"{dtype} {D} {T}")
        if eight:
            check_packed(packed, args)


# ---------------------------------------------------------------------------
# lengths on tensor copies
# ---------------------------------------------------------------------------
LENGTHS = [
    [512],
    [513],
    [640, 64, 0, 64, 128],
    [0, 3, 0, 0, 700, 64, 0],
    [1] * 600,
    [63, 1, 64, 2, 62, 500],
    [33 * 64 + 5, 3],
    [20 * 64, 1, 31 * 64, 17],
]


@pytest.mark.parametrize("lens", LENGTHS, ids=lambda v: "x".join(map(str, v[:4])) + f"n{len(v)}")
def test_lengths_on_tensor_copies(gdn, lens):
    args = inputs(lens, 128, BF16, sum(lens) + len(lens), slow=True)
    cu = cumulative(lens)
    d = dev(args)
    got, head = forward(gdn, d, cu)
    assert head is None or head[1] == 8
    check_forward(got, args, cu, str(lens[:5]))
    d_out, d_final = grads_of(lens, 128, BF16, 9)
    g, head = backward(gdn, d, cu, d_out.cuda(), d_final.cuda())
    assert head[1] == 8
    check_gradients(g, ref.backward(*args, cu.tolist(), d_out, d_final), BF16, str(lens[:5]))


# ---------------------------------------------------------------------------
# chunks joined through the workspace: types, widths, 8-bit copies
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("D,fused", [(1, False), (33, True), (128, False), (136, False), (260, False)])
@pytest.mark.parametrize("eight", [False, True])
def test_types_and_widths_over_many_chunks(gdn, dtype, D, fused, eight):
    """128 and 136 channels side by side are fetched by tensor copies (the 8-bit
    136 are not), 260 of a 4-byte type too; the rest row by row, or directly."""
    lens = [700, 0, 5, 841]
    args = inputs(lens, D, dtype, D, fused=fused)
    cu = cumulative(lens)
    d = dev(args)
    _, head = forward(gdn, d, cu)
    assert head is not None and head[1] == 8
    leaves = [t.detach().requires_grad_(True) for t in d]
    out, final = gdn.recurrence.run_autograd(*leaves, cu.cuda(), checkpoint="int8" if eight else None)
    check_forward((out.detach(), final.detach()), args, cu, f"{dtype} D={D}")
    if eight:
        check_packed(out.grad_fn.saved_tensors[3], args)
    d_out, d_final = grads_of(lens, D, dtype, 9)
    grads = torch.autograd.grad((out, final), leaves, (d_out.cuda(), d_final.cuda()))
    check_gradients(dict(zip(NAMES, grads)), ref.backward(*args, cu.tolist(), d_out, d_final, eight), dtype,
                    f"{dtype} D={D} eight={eight}")


def check_packed(packed, args):
    """The 8-bit x, a, b that the forward kept, bit for bit."""
    T, D = args[0].shape
    packed = packed.cpu()
    groups = -(-D // 128)
    values = packed[:3 * T * D].view(torch.int8).view(3, T, D).double()
    E = packed[3 * T * D:3 * T * (D + groups)].view(3, T, groups).int()
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), (E - 127).double()).repeat_interleave(128, -1)[..., :D]
    for w, t in enumerate((args[0], args[3], args[5])):
        assert torch.equal(values[w] * unit[w], ref.quantise(t)), "xab"[w]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("D", [64, 128, 136, 192, 260])
@pytest.mark.parametrize("T", [100, 900])
def test_packed_special_groups(gdn, dtype, D, T):
    """Groups at both ends of the type's range, of zeros, and with equal
    magnitudes, in the forward's own 8-bit copies."""
    g = torch.Generator().manual_seed(D + T)
    t = [torch.randn(T, D, generator=g).to(dtype) for _ in range(3)]
    for k in t:
        k[3] = 0
        k[5] *= torch.finfo(dtype).smallest_normal
        k[9, D // 2] = torch.finfo(dtype).max / 4
        k[11, -1] = 127.0
        k[12, 0] = -127.5
        k[17] = 1.0
    x, a, b = t
    p = torch.zeros(D)
    leaves = [v.cuda().requires_grad_(True) for v in (x, p, a, p.clone(), b)]
    out, _ = gdn.recurrence.run_autograd(leaves[0], None, *leaves[1:], checkpoint="int8")
    check_packed(out.grad_fn.saved_tensors[3], (x, None, p, a, p, b))


# ---------------------------------------------------------------------------
# groups of one
# ---------------------------------------------------------------------------
MANY = [90, 131, 64, 40, 257, 3, 128, 77, 150, 301, 20, 66, 5, 199, 64, 100]


@pytest.mark.parametrize("dtype,D,eight", [(BF16, 2048, False), (BF16, 2048, True), (FP16, 2048, False),
                                           (FP32, 1024, False), (BF16, 2050, False), (FP16, 2050, True),
                                           (FP32, 1030, True)])
def test_groups_of_one(gdn, dtype, D, eight):
    """Wide layers and several sequences: a state is published for each chunk,
    and streams are cut at starts that lie inside chunks."""
    args = inputs(MANY, D, dtype, D, slow=True)
    cu = cumulative(MANY)
    d = dev(args)
    got, head = forward(gdn, d, cu)
    assert head[0] > 4 and head[1] == 1, head
    check_forward(got, args, cu, f"{dtype} {D}")
    d_out, d_final = grads_of(MANY, D, dtype, 9)
    if not eight:
        g, head = backward(gdn, d, cu, d_out.cuda(), d_final.cuda())
        assert head[0] > 4 and head[1] == 1, head
        check_gradients(g, ref.backward(*args, cu.tolist(), d_out, d_final), dtype, f"{dtype} {D}")
        return
    leaves = [t.detach().requires_grad_(True) for t in d]
    out, final = gdn.recurrence.run_autograd(*leaves, cu.cuda(), checkpoint="int8")
    assert torch.equal(out, got[0]) and torch.equal(final, got[1])
    check_packed(out.grad_fn.saved_tensors[3], args)
    grads = torch.autograd.grad((out, final), leaves, (d_out.cuda(), d_final.cuda()))
    check_gradients(dict(zip(NAMES, grads)), ref.backward(*args, cu.tolist(), d_out, d_final, True), dtype,
                    f"{dtype} {D} 8 bits")


def test_groups_of_one_in_a_dense_batch_and_in_place(gdn):
    N, S, D = 6, 200, 2048
    args = inputs([S] * N, D, BF16, 4, slow=True)
    cu = cumulative([S] * N)
    x, state, A_log, a, dt_bias, b = dev(args)
    _, head = forward(gdn, [x, state, A_log, a, dt_bias, b], cu)
    assert head[1] == 1, head
    x, a, b = (t.view(N, S, D) for t in (x, a, b))
    out, final = gdn.recurrence.run(x, state, A_log, a, dt_bias, b)
    check_forward((out.view(-1, D), final), args, cu, "dense")
    slots = torch.tensor([4, 1, 0, 7, 3, 6], dtype=torch.int32, device="cuda")
    pool = torch.full((9, D), 5.0, device="cuda")
    pool[slots.long()] = state
    assert torch.equal(gdn.recurrence.run_pool(x, pool, slots, A_log, a, dt_bias, b), out)
    assert torch.equal(pool[slots.long()], final) and bool((pool[[2, 5, 8]] == 5.0).all())


@pytest.mark.parametrize("used", [1299, 700, 64, 0])
def test_rows_behind_in_groups_of_one(gdn, used):
    """Padded rows where states are published chunk by chunk."""
    lens = [used // 8] * 7 + [used - 7 * (used // 8)]
    T, D = 1300, 2048
    args = inputs(lens, D, BF16, used, rows=T)
    for i in (0, 3, 5):
        args[i][used:] = float("nan")
    cu = cumulative(lens)
    d = dev(args)
    out, final = gdn.recurrence.run(*d, cu.cuda())
    part = [t[:used] if i in (0, 3, 5) else t for i, t in enumerate(args)]
    check_forward((out[:used], final), part, cu, "padded")
    assert not out[used:].any()
    d_out, d_final = torch.randn(T, D, generator=torch.Generator().manual_seed(1)).to(BF16), torch.ones(8, D)
    d_out[used:] = float("nan")
    g = gdn.recurrence.backward(*d, cu.cuda(), d_out.cuda(), d_final.cuda())
    for n in ("dx", "da", "db"):
        assert not g[n][used:].any(), n
        g[n] = g[n][:used]
    check_gradients(g, ref.backward(*part, cu.tolist(), d_out[:used], d_final), BF16, "padded")
