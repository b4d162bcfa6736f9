"""The channelwise gated linear recurrence on the GPU against its definition in
float64, token by token, within bounds that count the roundings of fp32
(recurrence_ref.py), at the sizes, layouts and values where it can go wrong."""
import pytest
import torch

import recurrence_ref as ref

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _clean_status(gdn):
    gdn._native.read_device_status()
    yield
    assert gdn._native.read_device_status() == 0


def cumulative(lens):
    return torch.tensor([0, *lens], dtype=torch.int64).cumsum(0)


def inputs(lens, D, dtype, seed, with_state=True, slow=False, fused=False, rows=None):
    """x, state, A_log, a, dt_bias, b on the CPU (rows: T, if more than the lengths' sum)."""
    g = torch.Generator().manual_seed(seed)
    T = sum(lens) if rows is None else rows

    def act():
        return torch.randn(T, D, generator=g).to(dtype)

    if fused:
        joint = torch.randn(T, 3 * D + 5, generator=g).to(dtype)
        x, a, b = joint[:, :D], joint[:, D:2 * D], joint[:, 2 * D:3 * D]
    else:
        x, a, b = act(), act(), act()
    A_log = torch.rand(D, generator=g) * (3.0 if slow else 7.7) - 5.0
    dt_bias = torch.randn(D, generator=g) * 0.1
    state = torch.randn(len(lens), D, generator=g) if with_state else None
    return x, state, A_log, a, dt_bias, b


def dev(args):
    """On the GPU, in the same layout."""
    def move(t):
        if t is None:
            return None
        if t.dim() == 2 and t.stride(0) > t.shape[1] and t.shape[0] > 1:     # a part of wider rows
            wide = torch.empty(t.shape[0], t.stride(0), dtype=t.dtype, device="cuda")
            wide[:, :t.shape[1]] = t.cuda()
            return wide[:, :t.shape[1]]
        return t.cuda()
    return [move(t) for t in args]


def check_forward(got, args, cu, what):
    want = ref.forward(*args, cu.tolist())
    out, final = got
    ref.assert_close(out[:int(cu[-1])], tuple(v[:int(cu[-1])] for v in want["out"]), f"{what} out", out.dtype)
    ref.assert_close(final, want["final_state"], f"{what} final_state")


LENGTHS = [
    [1],
    [7],
    [64],                       # one chunk
    [65],
    [256],                      # the most rows that one launch takes
    [257],
    [0, 3, 0, 0, 70, 64, 0],    # empty sequences first, between and last
    [1] * 90,                   # a start and an end at every token
    [64, 64, 128, 64],          # starts on chunk boundaries
    [63, 1, 64, 2, 62, 200],
    [33 * 64 + 5, 3],           # a chain over more than one group of chunks
    [70 * 64, 1, 31 * 64, 17],
]


@pytest.mark.parametrize("lens", LENGTHS, ids=lambda v: "x".join(map(str, v[:4])) + f"n{len(v)}")
@pytest.mark.parametrize("with_state", [True, False])
def test_prefill_lengths(gdn, lens, with_state):
    args = inputs(lens, 132, BF16, sum(lens) + len(lens), with_state, slow=True)
    cu = cumulative(lens)
    check_forward(gdn.recurrence.run(*dev(args), cu.cuda()), args, cu, str(lens[:5]))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("D", [1, 3, 4, 33, 128, 129, 260])
@pytest.mark.parametrize("fused", [False, True])
def test_prefill_types_and_widths(gdn, dtype, D, fused):
    lens = [300, 5, 41]
    args = inputs(lens, D, dtype, D, fused=fused)
    cu = cumulative(lens)
    check_forward(gdn.recurrence.run(*dev(args), cu.cuda()), args, cu, f"{dtype} D={D}")


@pytest.mark.parametrize("shape", [(3, 1), (2, 64), (5, 77), (1, 400), (70, 9)])
def test_prefill_dense_equals_packed(gdn, shape):
    N, S = shape
    args = inputs([S] * N, 96, BF16, N * S)
    d = dev(args)
    out, final = gdn.recurrence.run(*d, cumulative([S] * N).cuda())
    x, state, A_log, a, dt_bias, b = d
    out2, final2 = gdn.recurrence.run(x.view(N, S, 96), state, A_log, a.view(N, S, 96), dt_bias, b.view(N, S, 96))
    assert torch.equal(out, out2.view_as(out)) and torch.equal(final, final2)
    check_forward((out, final), args, cumulative([S] * N), f"dense {shape}")


def test_one_sequence_without_cu_seqlens(gdn):
    args = inputs([130], 64, BF16, 2)
    cu = cumulative([130])
    check_forward(gdn.recurrence.run(*dev(args)), args, cu, "one")


def test_nothing_to_do(gdn):
    d = dev(inputs([0, 0], 40, BF16, 1))
    out, final = gdn.recurrence.run(*d, torch.zeros(3, dtype=torch.int64, device="cuda"))
    assert out.shape == (0, 40) and torch.equal(final, d[1])
    out, final = gdn.recurrence.run(d[0], None, *d[2:], torch.zeros(3, dtype=torch.int64, device="cuda"))
    assert torch.equal(final, torch.zeros(2, 40, device="cuda"))
    out, final = gdn.recurrence.run(d[0].view(2, 0, 40), d[1], d[2], d[3].view(2, 0, 40), d[4], d[5].view(2, 0, 40))
    assert torch.equal(final, d[1])


@pytest.mark.parametrize("lens", [[0] * 1100, [0] * 600 + [5] + [0] * 600, [0, 1, 0, 2] * 500])
def test_many_sequences_most_of_them_empty(gdn, lens):
    args = inputs(lens, 24, BF16, 77)
    cu = cumulative(lens)
    check_forward(gdn.recurrence.run(*dev(args), cu.cuda()), args, cu, "empty")
    d_final = torch.randn(len(lens), 24, generator=torch.Generator().manual_seed(1))
    d_out = torch.randn(sum(lens), 24, generator=torch.Generator().manual_seed(2)).to(BF16)
    got = gdn.recurrence.backward(*dev(args), cu.cuda(), d_out.cuda(), d_final.cuda())
    check_gradients(got, ref.backward(*args, cu.tolist(), d_out, d_final), BF16, "empty")


@pytest.mark.parametrize("T", [100, 1000])
def test_state_updated_in_place_and_continued(gdn, T):
    """A sequence cut in two, the second part continued from the state that the
    first left in place, gives the whole's outputs."""
    lens = [T, T // 3]
    args = inputs(lens, 128, FP32, T, slow=True)
    cu = cumulative(lens)
    x, state, A_log, a, dt_bias, b = dev(args)
    s = state.clone()
    outs = []
    for lo, hi in ((0, T // 2), (T // 2, T)):
        rows = torch.cat([torch.arange(lo, hi), T + torch.arange(lo // 3, hi // 3)])
        c = cumulative([hi - lo, hi // 3 - lo // 3]).cuda()
        out = torch.empty(len(rows), 128, device="cuda")
        ws = gdn.recurrence.alloc_workspace(len(rows), 128, "cuda")
        gdn.recurrence.run_into(x[rows], s, A_log, a[rows], dt_bias, b[rows], c, out, s, ws)
        outs.append((rows, out))
    whole = torch.empty_like(x)
    for rows, out in outs:
        whole[rows] = out
    check_forward((whole, s), args, cu, "continued")


@pytest.mark.parametrize("lens", [[20, 0, 9], [500, 0, 300, 64]])
def test_pool_equals_dense_states(gdn, lens):
    args = inputs(lens, 72, BF16, 5)
    x, state, A_log, a, dt_bias, b = dev(args)
    cu = cumulative(lens).cuda()
    out, final = gdn.recurrence.run(x, state, A_log, a, dt_bias, b, cu)
    P = len(lens) + 4
    slots = torch.randperm(P, generator=torch.Generator().manual_seed(3))[:len(lens)].to(torch.int32).cuda()
    pool = torch.randn(P, 72, device="cuda")
    pool[slots.long()] = state
    before = pool.clone()
    got = gdn.recurrence.run_pool(x, pool, slots, A_log, a, dt_bias, b, cu)
    assert torch.equal(got, out) and torch.equal(pool[slots.long()], final)
    others = [i for i in range(P) if i not in slots.tolist()]
    assert torch.equal(pool[others], before[others])


@pytest.mark.parametrize("lens", [[5000, 100, 37, 3000, 65, 1], [70] * 60, [1000, 7000], [33] * 7 + [3000]])
def test_states_in_place_where_chunks_are_cut(gdn, lens):
    """Sequences that start inside a chunk where the rows are cut into streams:
    the later stream may finish such a sequence, and overwrite its state, before
    the earlier one has come to the chunk where it starts."""
    for D in (64, 512):
        x, state, A_log, a, dt_bias, b = dev(inputs(lens, D, BF16, 13, slow=True))
        cu = cumulative(lens).cuda()
        out, final = gdn.recurrence.run(x, state, A_log, a, dt_bias, b, cu)
        slots = torch.randperm(len(lens), generator=torch.Generator().manual_seed(3)).to(torch.int32).cuda()
        for _ in range(4):
            pool = torch.empty_like(state)
            pool[slots.long()] = state
            assert torch.equal(gdn.recurrence.run_pool(x, pool, slots, A_log, a, dt_bias, b, cu), out)
            assert torch.equal(pool[slots.long()], final)


@pytest.mark.parametrize("T,used", [(100, 37), (256, 0), (900, 512), (900, 70)])
def test_rows_behind_the_last_sequence(gdn, T, used):
    """Padded rows, NaN in all inputs there, are left alone by the _into form
    and zero in what `run` and `backward` return."""
    lens = [used // 2, used - used // 2]
    args = inputs(lens, 136, BF16, T + used, rows=T)
    for i in (0, 3, 5):
        args[i][used:] = float("nan")
    cu = cumulative(lens)
    d = dev(args)
    out = torch.full((T, 136), 7.0, dtype=BF16, device="cuda")
    final = torch.empty(2, 136, device="cuda")
    gdn.recurrence.run_into(*d, cu.cuda(), out, final, gdn.recurrence.alloc_workspace(T, 136, "cuda"))
    assert bool((out[used:] == 7.0).all())
    part = [t[:used] if i in (0, 3, 5) else t for i, t in enumerate(args)]
    check_forward((out[:used], final), part, cu, "padded")
    out2, final2 = gdn.recurrence.run(*d, cu.cuda())
    assert torch.equal(out2[:used], out[:used]) and torch.equal(final2, final) and not out2[used:].any()
    d_out = torch.randn(T, 136, generator=torch.Generator().manual_seed(1)).to(BF16)
    d_out[used:] = float("nan")
    g = gdn.recurrence.backward(*d, cu.cuda(), d_out.cuda())
    for n in ("dx", "da", "db"):
        assert not g[n][used:].any(), n
    want = ref.backward(*part, cu.tolist(), d_out[:used], None)
    check_gradients({k: v if k not in ("dx", "da", "db") else v[:used] for k, v in g.items()}, want, BF16, "padded")


# ---------------------------------------------------------------------------
# values
# ---------------------------------------------------------------------------
def test_extreme_gates(gdn):
    """Gates that forget everything, nothing, and inputs far out in both
    directions: same limits as the formula's."""
    big = [0.0, 1.0, -1.0, 15.0, -15.0, 90.0, -90.0, 1e4, -1e4, float("inf"), -float("inf")]
    T, D = 90, len(big)
    x = torch.randn(T, D, generator=torch.Generator().manual_seed(4))
    a = torch.tensor(big).repeat(T, 1)
    b = torch.tensor(big[::-1]).repeat(T, 1)
    A_log = torch.linspace(-6, 2, D)
    dt_bias = torch.zeros(D)
    state = torch.randn(1, D, generator=torch.Generator().manual_seed(5))
    out, final = gdn.recurrence.run(*dev((x, state, A_log, a, dt_bias, b)))
    z = a.double()
    g = torch.exp(-A_log.double().exp() * torch.logaddexp(z, torch.zeros_like(z)))
    u = torch.sigmoid(b.double()) * x.double()
    h = state.double()[0]
    for t in range(T):
        h = g[t] * h + u[t]
        # exp(-90) and less may be rounded to zero; elsewhere the relative
        # error of a gate is at most |lg| 300 u, far below 1e-4 of the terms
        torch.testing.assert_close(out[t].double().cpu(), h, rtol=1e-4, atol=1e-4)
    assert torch.isfinite(final).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("lens", [[30, 40, 20], [1000, 64 * 40, 777]])
def test_non_finite_values_stay_in_their_sequence_and_channel(gdn, bad, lens):
    args = inputs(lens, 130, BF16, 8)
    s = lens[0]
    args[0][s + 3, 5] = bad
    args[3][s + lens[1] // 2, 77] = float("nan")
    args[1][1, 100] = bad
    d = dev(args)
    cu = cumulative(lens)
    out, final = gdn.recurrence.run(*d, cu.cuda())
    clean = [t.clone() if t is not None else None for t in args]
    clean[0][s + 3, 5] = 0
    clean[3][s + lens[1] // 2, 77] = 0
    clean[1][1, 100] = 0
    cout, cfinal = gdn.recurrence.run(*dev(clean), cu.cuda())
    touched = torch.zeros(sum(lens), 130, dtype=torch.bool)
    touched[s + 3:s + lens[1], 5] = touched[s + lens[1] // 2:s + lens[1], 77] = True
    touched[s:s + lens[1], 100] = True
    same = (out == cout).cpu()
    assert bool(same[~touched].all())
    assert not torch.isfinite(out[s + 3, 5]) and torch.isnan(out[s + lens[1] - 1, 77])
    assert torch.equal(final[0], cfinal[0]) and torch.equal(final[2], cfinal[2])


def test_long_memory_keeps_its_precision(gdn):
    """Gates within 1e-3 of one over 20,000 tokens: the rounding of the gates
    adds up, and no more than the bound."""
    lens = [20000]
    g = torch.Generator().manual_seed(6)
    D = 8
    x, a, b = (torch.randn(20000, D, generator=g) for _ in range(3))
    A_log, dt_bias = torch.full((D,), -1.0), torch.full((D,), -7.0)
    args = (x, torch.randn(1, D, generator=g), A_log, a, dt_bias, b)
    check_forward(gdn.recurrence.run(*dev(args)), args, cumulative(lens), "long")


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (1, 1, 1024), (3, 1, 130), (5, 4, 36), (2, 64, 129), (300, 2, 128)])
@pytest.mark.parametrize("fused", [False, True])
def test_decode(gdn, dtype, B, T, D, fused):
    args = inputs([T] * B, D, dtype, B + T + D, fused=fused)
    cu = cumulative([T] * B)
    x, state, A_log, a, dt_bias, b = dev(args)
    if T > 1:
        x, a, b = (t.unflatten(0, (B, T)) for t in (x, a, b))
    out, new = gdn.recurrence.decode(x, state, A_log, a, dt_bias, b)
    check_forward((out.reshape(B * T, D), new), args, cu, "decode")
    out2, new2, inter = gdn.recurrence.decode(x, state, A_log, a, dt_bias, b, return_intermediate=True)
    assert torch.equal(out, out2) and torch.equal(new, new2)
    assert torch.equal(inter[:, -1], new) and torch.equal(inter.to(dtype).view(out.shape), out)
    s = state.clone()
    assert torch.equal(gdn.recurrence.decode_inplace(x, s, A_log, a, dt_bias, b), out) and torch.equal(s, new)
    slots = torch.randperm(B + 3, generator=torch.Generator().manual_seed(1))[:B].to(torch.int32).cuda()
    pool = torch.zeros(B + 3, D, device="cuda")
    pool[slots.long()] = state
    assert torch.equal(gdn.recurrence.decode_pool(x, pool, slots, A_log, a, dt_bias, b), out)
    assert torch.equal(pool[slots.long()], new)
    zero, nz = gdn.recurrence.decode(x, None, A_log, a, dt_bias, b)
    part = (args[0], None, *args[2:])
    check_forward((zero.reshape(B * T, D), nz), part, cu, "decode from zeros")


def test_prefill_then_decode_as_one_sequence(gdn):
    """A serving run: prompts prefilled into the pool, then tokens decoded one
    and four at a time, against the recurrence over all of them."""
    lens, steps = [200, 3, 77], [1, 1, 4]
    total = [n + sum(steps) for n in lens]
    args = inputs(total, 96, BF16, 12, slow=True)
    want = ref.forward(*args, cumulative(total).tolist())["out"]
    x, state, A_log, a, dt_bias, b = dev(args)
    starts = cumulative(total)[:-1]
    pool = torch.zeros(8, 96, device="cuda")
    slots = torch.tensor([6, 1, 3], dtype=torch.int32, device="cuda")
    pool[slots.long()] = state
    rows = torch.cat([torch.arange(s, s + n) for s, n in zip(starts.tolist(), lens)])
    out = torch.empty_like(x)
    out[rows] = gdn.recurrence.run_pool(x[rows], pool, slots, A_log, a[rows], dt_bias, b[rows],
                                        cumulative(lens).cuda())
    at = starts + torch.tensor(lens)
    for n in steps:
        rows = at[:, None] + torch.arange(n)
        out[rows.flatten()] = gdn.recurrence.decode_pool(x[rows], pool, slots, A_log, a[rows], dt_bias,
                                                         b[rows]).flatten(0, 1)
        at = at + n
    ref.assert_close(out, want, "serving run", BF16)


# ---------------------------------------------------------------------------
# backward
# ---------------------------------------------------------------------------
def check_gradients(got, want, dtype, what):
    for name, value in want.items():
        if got[name] is None:
            continue
        ref.assert_close(got[name], value, f"{what} {name}", dtype if name in ("dx", "da", "db") else None)


@pytest.mark.parametrize("lens", LENGTHS, ids=lambda v: "x".join(map(str, v[:4])) + f"n{len(v)}")
@pytest.mark.parametrize("final", [True, False])
def test_backward_lengths(gdn, lens, final):
    args = inputs(lens, 132, BF16, sum(lens) + len(lens), slow=True)
    cu = cumulative(lens)
    g = torch.Generator().manual_seed(9)
    d_out = torch.randn(sum(lens), 132, generator=g).to(BF16)
    d_final = torch.randn(len(lens), 132, generator=g) if final else None
    got = gdn.recurrence.backward(*dev(args), cu.cuda(), d_out.cuda(), None if d_final is None else d_final.cuda())
    check_gradients(got, ref.backward(*args, cu.tolist(), d_out, d_final), BF16, str(lens[:5]))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("D", [1, 4, 33, 128, 260])
@pytest.mark.parametrize("eight", [False, True])
def test_autograd_types_and_widths(gdn, dtype, D, eight):
    lens = [300, 0, 5, 141]
    args = inputs(lens, D, dtype, D, fused=True)
    cu = cumulative(lens)
    g = torch.Generator().manual_seed(9)
    d_out = torch.randn(sum(lens), D, generator=g).to(dtype)
    d_final = torch.randn(len(lens), D, generator=g)
    leaves = [t.detach().requires_grad_(True) for t in dev(args)]
    out, final = gdn.recurrence.run_autograd(*leaves, cu.cuda(), checkpoint="int8" if eight else None)
    check_forward((out.detach(), final.detach()), args, cu, "autograd")
    grads = torch.autograd.grad((out, final), leaves, (d_out.cuda(), d_final.cuda()))
    names = ("dx", "d_state", "dA_log", "da", "ddt_bias", "db")
    for leaf, grad in zip(leaves, grads):
        assert grad.dtype == leaf.dtype and grad.shape == leaf.shape
    check_gradients(dict(zip(names, grads)), ref.backward(*args, cu.tolist(), d_out, d_final, eight), dtype,
                    f"{dtype} D={D} eight={eight}")


@pytest.mark.parametrize("eight", [False, True])
def test_autograd_dense_without_state_and_partial_gradients(gdn, eight):
    N, S, D = 3, 150, 68
    args = inputs([S] * N, D, BF16, 3, with_state=False)
    x, _, A_log, a, dt_bias, b = dev(args)
    x, a, b = (t.view(N, S, D) for t in (x, a, b))
    a.requires_grad_(True)
    A_log.requires_grad_(True)
    out, final = gdn.recurrence.run_autograd(x, None, A_log, a, dt_bias, b, checkpoint="int8" if eight else None)
    d_out = torch.randn(N, S, D, generator=torch.Generator().manual_seed(2)).to(BF16)
    (out * d_out.cuda()).sum().backward()                 # final_state unused
    want = ref.backward(*args, cumulative([S] * N).tolist(), d_out.view(-1, D), None, eight)
    ref.assert_close(a.grad.view(-1, D), want["da"], "da", BF16)
    ref.assert_close(A_log.grad, want["dA_log"], "dA_log")
    # only the final state is used: d_out is zero
    out, final = gdn.recurrence.run_autograd(x, None, A_log, a, dt_bias, b, checkpoint="int8" if eight else None)
    d_final = torch.randn(N, D, generator=torch.Generator().manual_seed(3))
    got, = torch.autograd.grad(final, a, d_final.cuda())
    want = ref.backward(*args, cumulative([S] * N).tolist(), torch.zeros(N * S, D, dtype=BF16), d_final, eight)
    ref.assert_close(got.view(-1, D), want["da"], "da from the final state", BF16)


def test_gradient_of_expanded_inputs(gdn):
    """One row of gate inputs for all tokens (stride 0), and a d_out that is
    one number: the gradients sum over the uses."""
    T, D = 200, 40
    g = torch.Generator().manual_seed(7)
    x, a1, b = (torch.randn(T, D, generator=g).cuda(), torch.randn(1, D, generator=g).cuda(),
                torch.randn(T, D, generator=g).cuda())
    A_log, dt_bias = torch.zeros(D, device="cuda"), torch.zeros(D, device="cuda")
    a1.requires_grad_(True)
    out, _ = gdn.recurrence.run_autograd(x, None, A_log, a1.expand(T, D), dt_bias, b)
    out.sum().backward()
    want = ref.backward(x.cpu(), None, A_log.cpu(), a1.detach().cpu().expand(T, D), dt_bias.cpu(), b.cpu(), [0, T],
                        torch.ones(T, D), None)
    value, bound = want["da"]
    # torch's sum over T rows: at most T roundings of partial sums
    ref.assert_close(a1.grad, (value.sum(0, keepdim=True),
                               bound.sum(0, keepdim=True) + T * ref.U * value.abs().sum(0, keepdim=True)), "da")


def test_gradients_against_differences(gdn):
    """Directional derivative of a loss of the kernel's own fp32 outputs by
    central differences.  With steps e and e / 2 combined (error e^4) at
    e = 2^-4 what is left is the rounding of the outputs, about 1e-6 of the
    loss's terms over 2 e; 2e-3 of the derivative's terms covers both."""
    lens = [70, 130]
    args = inputs(lens, 24, FP32, 21)
    cu = cumulative(lens).cuda()
    d = dev(args)
    g = torch.Generator().manual_seed(22)
    w_out, w_fin = torch.randn(200, 24, generator=g).cuda(), torch.randn(2, 24, generator=g).cuda()
    grads = gdn.recurrence.backward(*d, cu, w_out, w_fin)
    names = ("dx", "d_state", "dA_log", "da", "ddt_bias", "db")

    def loss(i, v, s):
        moved = [t + s * v if k == i else t for k, t in enumerate(d)]
        out, fin = gdn.recurrence.run(*moved, cu)
        return (out.double() * w_out).sum() + (fin.double() * w_fin).sum()

    for i, name in enumerate(names):
        v = torch.randn(d[i].shape, generator=g).cuda()
        e = 2.0 ** -4
        d1 = (loss(i, v, e) - loss(i, v, -e)) / (2 * e)
        d2 = (loss(i, v, e / 2) - loss(i, v, -e / 2)) / e
        want = (4 * d2 - d1) / 3
        got = (grads[name].double() * v).sum()
        scale = (grads[name].double() * v).abs().sum()
        assert abs(got - want) <= 2e-3 * scale, (name, got.item(), want.item(), scale.item())


def test_results_are_the_same_bits_on_every_run(gdn):
    lens = [64 * 300 + 3, 5000, 1, 0, 777]
    args = dev(inputs(lens, 384, BF16, 31, slow=True))
    cu = cumulative(lens).cuda()
    d_out = torch.randn(sum(lens), 384, device="cuda").to(BF16)
    first = None
    for _ in range(5):
        out, final = gdn.recurrence.run(*args, cu)
        g = gdn.recurrence.backward(*args, cu, d_out)
        now = [out, final, *(g[k] for k in sorted(g))]
        first = first or now
        assert all(torch.equal(p, q) for p, q in zip(first, now))


# ---------------------------------------------------------------------------
# streams, graphs, refusals
# ---------------------------------------------------------------------------
def test_two_streams_at_once(gdn):
    lens = [6000, 3000]
    cu = cumulative(lens).cuda()
    sets = [dev(inputs(lens, 256, BF16, s)) for s in (41, 42)]
    want = [gdn.recurrence.run(*s, cu) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(gdn.recurrence.run(*s, cu))
        torch.cuda.synchronize()
        for p, q in zip(want, got):
            assert torch.equal(p[0], q[0]) and torch.equal(p[1], q[1])


def test_calls_from_a_thread_that_has_not_used_cuda(gdn):
    """As autograd's threads are: with all memory from torch's cache nothing
    before the call makes the device's context current there."""
    import threading
    import cases
    from gpu_util import prefill_args

    d = dev(inputs([600], 128, BF16, 71))
    d_out = torch.randn(600, 128, device="cuda").to(BF16)
    want = gdn.recurrence.backward(*d, None, d_out)
    out, final = gdn.recurrence.run(*d)
    out2, final2 = torch.empty_like(out), torch.empty_like(final)
    ws = gdn.recurrence.alloc_workspace(600, 128, "cuda")
    g = {k: torch.empty_like(v) for k, v in want.items()}
    bws = gdn.recurrence.alloc_backward_workspace(600, 128, "cuda")
    p = prefill_args(cases.prefill_inputs(seed=3, lens=[100, 30], with_state=True))
    p_out, p_final = gdn.prefill.run(*p, None)
    p_out2, p_final2 = torch.empty_like(p_out), torch.empty_like(p_final)
    pws = gdn.prefill.alloc_workspace(130, 2, "cuda")
    stream = torch.cuda.current_stream().cuda_stream
    errors = []

    def call(f):
        try:
            f()
        except Exception as e:      # noqa: BLE001  (reported by the test's own thread)
            errors.append(e)

    for f in (lambda: gdn.recurrence.run_into(*d, None, out2, final2, ws, stream=stream),
              lambda: gdn.recurrence.backward_into(*d, None, d_out, None, g["dx"], g["da"], g["db"], g["dA_log"],
                                                   g["ddt_bias"], g["d_state"], bws, stream=stream),
              lambda: gdn.prefill.prefill_into(*p, None, p_out2, p_final2, pws, stream=stream)):
        t = threading.Thread(target=call, args=(f,))
        t.start()
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    assert torch.equal(out, out2) and torch.equal(final, final2)
    assert torch.equal(p_out, p_out2) and torch.equal(p_final, p_final2)
    for k, v in want.items():
        assert torch.equal(v, g[k]), k


def test_captured_training_step_with_new_lengths_on_replay(gdn):
    """Forward and backward in a graph; replays see other values and other
    cu_seqlens, fewer rows among them."""
    T, D = 700, 128
    args = dev(inputs([300, 400], D, BF16, 51))
    cu = cumulative([300, 400]).cuda()
    leaves = [t.detach().requires_grad_(True) for t in args]
    d_out = torch.randn(T, D, device="cuda").to(BF16)

    def step():
        out, final = gdn.recurrence.run_autograd(*leaves, cu, checkpoint="int8")
        grads = torch.autograd.grad(out, leaves, d_out)
        return (out.detach(), final.detach(), *grads)      # no graph of the leaves outlives the step

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for lens in ([300, 400], [1, 650], [0, 699]):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(T, D, device="cuda").to(BF16))
            cu.copy_(cumulative(lens))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        for p, q in zip(got, want):
            assert torch.equal(p, q), lens


@pytest.mark.parametrize("cu,rows", [([0, 60, 40], 100), ([1, 60, 100], 100), ([0, 60, 101], 100),
                                     ([0, 500, 400, 700], 700), ([0, 800, 700], 700)])
def test_bad_seqlens_write_nothing(gdn, cu, rows):
    args = dev(inputs([1] * (len(cu) - 1), 64, BF16, 1, rows=rows))
    c = torch.tensor(cu, dtype=torch.int64, device="cuda")
    out = torch.full((rows, 64), 3.0, dtype=BF16, device="cuda")
    final = torch.full((len(cu) - 1, 64), 3.0, device="cuda")
    gdn.recurrence.run_into(*args, c, out, final, gdn.recurrence.alloc_workspace(rows, 64, "cuda"))
    assert gdn._native.read_device_status() == 1
    assert bool((out == 3.0).all()) and bool((final == 3.0).all())
    g = {k: torch.full((rows, 64), 3.0, dtype=BF16, device="cuda") for k in ("dx", "da", "db")}
    p = {k: torch.full((64,), 3.0, device="cuda") for k in ("dA_log", "ddt_bias")}
    ds = torch.full_like(final, 3.0)
    gdn.recurrence.backward_into(*args, c, out, None, g["dx"], g["da"], g["db"], p["dA_log"], p["ddt_bias"], ds,
                                 gdn.recurrence.alloc_backward_workspace(rows, 64, "cuda"))
    assert gdn._native.read_device_status() == 1
    for t in (*g.values(), *p.values(), ds):
        assert bool((t == 3.0).all())


@pytest.mark.parametrize("rows", [50, 500])
def test_bad_slots(gdn, rows):
    lens = [rows // 2, rows - rows // 2]
    x, state, A_log, a, dt_bias, b = dev(inputs(lens, 64, BF16, 1))
    pool = torch.full((5, 64), 3.0, device="cuda")
    slots = torch.tensor([4, 5], dtype=torch.int32, device="cuda")
    out = torch.full((rows, 64), 3.0, dtype=BF16, device="cuda")
    gdn.recurrence.run_pool_into(x, pool, slots, A_log, a, dt_bias, b, cumulative(lens).cuda(), out,
                                 gdn.recurrence.alloc_workspace(rows, 64, "cuda"))
    assert gdn._native.read_device_status() == 3
    assert bool((out == 3.0).all()) and bool((pool == 3.0).all())
    # decode skips that request alone
    got = gdn.recurrence.decode_pool(x[:2], pool, slots, A_log, a[:2], dt_bias, b[:2])
    assert gdn._native.read_device_status() == 3
    assert bool((pool[:4] == 3.0).all()) and not bool((pool[4] == 3.0).all())
    want, _ = gdn.recurrence.decode(x[:1], torch.full((1, 64), 3.0, device="cuda"), A_log, a[:1], dt_bias, b[:1])
    assert torch.equal(got[:1], want)


def test_copied_layouts(gdn):
    """Channels that are not side by side, and batches with gaps, are copied."""
    args = inputs([50] * 4, 24, BF16, 61)
    x, state, A_log, a, dt_bias, b = dev(args)
    want, wf = gdn.recurrence.run(*(t.view(4, 50, 24) if t.shape[0] == 200 else t
                                    for t in (x, state, A_log, a, dt_bias, b)))
    apart = torch.zeros(4, 60, 24, dtype=BF16, device="cuda")[:, :50]
    apart.copy_(a.view(4, 50, 24))
    got, gf = gdn.recurrence.run(x.view(4, 50, 24).transpose(1, 2).contiguous().transpose(1, 2), state, A_log, apart,
                                 dt_bias, b.view(4, 50, 24))
    assert torch.equal(got, want) and torch.equal(gf, wf)
    with pytest.raises(ValueError, match="stream"):
        gdn.recurrence.run_into(x.view(4, 50, 24), state, A_log, apart, dt_bias, b.view(4, 50, 24), None,
                                torch.empty_like(want), torch.empty_like(wf),
                                gdn.recurrence.alloc_workspace(200, 24, "cuda"),
                                stream=torch.cuda.current_stream().cuda_stream)
