"""Cases for measuring the channelwise gated linear recurrence and the 8-bit activation checkpoints.

The recurrence keeps one fp32 state per channel and uses the gates of the GDN kernels, one per channel:
    g_t = exp(-exp(A_log) softplus(a_t + dt_bias)),  beta_t = sigmoid(b_t),  h_t = g_t h_{t-1} + beta_t x_t,  out_t = h_t.
It is measured as a decode step, as a prefill over packed sequences, and as a training step (forward and backward), the
latter also with the activations kept in 8 bits between the two.  The checkpoint format is measured alone as well
(pack and unpack): int8 in groups of 128 values of a row that share one power of two.

With `own` false the operators run in their plain form: elementary torch operations in fp32 (the recurrence as a
doubling scan).  With `own` true they are called as a user of this package calls them.
"""
from __future__ import annotations

import importlib
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GROUP = 128   # values of a row that share a scale in a packed checkpoint
TOP = {torch.bfloat16: 121, torch.float16: 9, torch.float32: 121}   # no larger scale, so that 127 2^e is finite in the type
CHUNK = 64    # packed tokens between two exact states that an 8-bit training step keeps


def _gdn():
    return importlib.import_module("track-c-gdn_b200")


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one request decoding one token: nothing but latency
        {"name": "decode-b1", "op": "decode", "type": "bf16", "batch": 1, "tokens": 1, "channels": 1024,
         "pool": 0, "fused": False},
        # the decode half of the mixed serving step: 4096 requests, their states in a pool
        {"name": "decode-pool-b4096", "op": "decode", "type": "bf16", "batch": 4096, "tokens": 1, "channels": 1024,
         "pool": 4608, "fused": True},
        # one short prompt
        {"name": "prefill-one-269", "op": "prefill", "type": "bf16", "lengths": "one", "count": 1, "longest": 269,
         "channels": 1024, "state": False, "fused": False},
        # a ragged batch that continues from states, with rows that no vector load fits
        {"name": "prefill-ragged-odd-fp16", "op": "prefill", "type": "fp16", "lengths": "uniform", "count": 32,
         "longest": 3000, "channels": 1021, "state": True, "fused": False},
        # the prefill half of the mixed serving step: 256 new sequences of 512 to 8192 tokens
        {"name": "prefill-mixed-256", "op": "prefill", "type": "bf16", "lengths": "mixed", "count": 256,
         "longest": 8192, "channels": 1024, "state": False, "fused": True},
        # one long document in fp32: all the parallelism there is lies along the tokens
        {"name": "prefill-long-fp32", "op": "prefill", "type": "fp32", "lengths": "one", "count": 1, "longest": 65536,
         "channels": 1024, "state": True, "fused": False},
        # a training step over one sequence
        {"name": "train-one-4096", "op": "train", "type": "bf16", "lengths": "one", "count": 1, "longest": 4096,
         "channels": 1024, "state": False, "fused": False},
        # a training step over a dense batch
        {"name": "train-dense-8x4096", "op": "train", "type": "bf16", "lengths": "dense", "count": 8, "longest": 4096,
         "channels": 2048, "state": False, "fused": False},
        # training on packed sequences with 8-bit checkpoints, states carried in and out
        {"name": "train8-ragged", "op": "train8", "type": "bf16", "lengths": "uniform", "count": 32, "longest": 3000,
         "channels": 1024, "state": True, "fused": True},
        # the dense batch with 8-bit checkpoints
        {"name": "train8-dense-8x4096", "op": "train8", "type": "bf16", "lengths": "dense", "count": 8,
         "longest": 4096, "channels": 2048, "state": False, "fused": False},
        # the q, k and v of one short prompt of the GDN prefill, packed and restored
        {"name": "pack-qkv-269", "op": "pack", "type": "bf16", "rows": 269, "heads": "4,4,8", "channels": 128},
        # the same for a training batch of 65536 tokens
        {"name": "pack-qkv-65536", "op": "pack", "type": "bf16", "rows": 65536, "heads": "4,4,8", "channels": 128},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "prefill", "prefill", "train", "train8", "pack"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    channels = _log_int(rng, 32, 4096)
    how = rng.random()
    if how < 0.6:                       # most layers are as wide as a few heads
        channels = max(128, channels // 128 * 128)
    elif how < 0.8:
        channels = max(32, channels // 8 * 8)
    fused = rng.random() < 0.4
    if op == "decode":
        batch = _log_int(rng, 1, 8192)
        tokens = rng.choice([1, 1, 1, 2, 4, 5])
        return {"op": op, "type": kind, "batch": batch, "tokens": tokens, "channels": channels,
                "pool": rng.choice([0, batch + batch // 8 + 1]), "fused": fused}
    if op == "pack":
        return {"op": op, "type": kind, "rows": _log_int(rng, 1, 1 << 17), "heads": rng.choice(["1", "8,8", "4,4,8"]),
                "channels": rng.choice([64, 128, 256, channels // 8 + 1])}
    lengths = rng.choice(["one", "uniform", "mixed", "dense"])
    count = 1 if lengths == "one" else _log_int(rng, 2, 256)
    room = (1 << 26) // channels        # tokens in all
    longest = _log_int(rng, 2, max(4, min(65536, room // count)))
    return {"op": op, "type": kind, "lengths": lengths, "count": count, "longest": longest, "channels": channels,
            "state": rng.random() < 0.5, "fused": fused}


def _lengths(case, seed):
    n, longest = case["count"], case["longest"]
    if case["lengths"] in ("one", "dense"):
        return [longest] * n
    low = 17 if case["lengths"] == "uniform" else 512
    low = min(low, max(1, longest // 16))
    # the same lengths for every seed: the case names its size, the seed its values
    return [int(v) for v in np.random.default_rng(4).integers(low, longest + 1, size=n)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _activations(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEVICE).to(dtype)


def _xab(g, lead, channels, dtype, fused):
    """x, a, b: three tensors, or the three parts of one projection's output."""
    if fused:
        joint = _activations(g, (*lead, 3 * channels), dtype)
        return [joint[..., i * channels:(i + 1) * channels] for i in range(3)]
    return [_activations(g, (*lead, channels), dtype) for _ in range(3)]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    dtype, C = TYPES[case["type"]], case["channels"]
    s = {"case": case, "own": own}
    if case["op"] == "pack":
        # activations of a few magnitudes, as the heads of a layer have them
        s["tensors"] = []
        for h in map(int, case["heads"].split(",")):
            size = torch.exp(torch.randn(h, 1, generator=g, device=DEVICE))
            s["tensors"].append((torch.randn(case["rows"], h, C, generator=g, device=DEVICE) * size).to(dtype))
        return s
    # decays from a few tokens' memory to some hundred
    s["A_log"] = torch.rand(C, generator=g, device=DEVICE) * 7.7 - 5.0
    s["dt_bias"] = torch.randn(C, generator=g, device=DEVICE) * 0.1
    if case["op"] == "decode":
        B, T = case["batch"], case["tokens"]
        s["x"], s["a"], s["b"] = _xab(g, (B,) if T == 1 else (B, T), C, dtype, case["fused"])
        P = case["pool"] or B
        s["state"] = torch.randn(P, C, generator=g, device=DEVICE)
        if case["pool"]:
            s["slots"] = torch.randperm(P, generator=g, device=DEVICE)[:B].to(torch.int32)
        return s
    lens = _lengths(case, seed)
    N, T = len(lens), sum(lens)
    dense = case["lengths"] == "dense"
    s["dense"], s["lens"], s["T"], s["N"] = dense, lens, T, N
    cu = torch.zeros(N + 1, dtype=torch.int64)
    cu[1:] = torch.tensor(lens).cumsum(0)
    s["cu"] = cu.to(DEVICE)
    lead = (N, lens[0]) if dense else (T,)
    s["x"], s["a"], s["b"] = _xab(g, lead, C, dtype, case["fused"])
    s["state"] = torch.randn(N, C, generator=g, device=DEVICE) if case["state"] else None
    if case["op"] == "prefill":
        if own:
            s["out"] = torch.empty(*lead, C, dtype=dtype, device=DEVICE)
            s["final"] = torch.empty(N, C, device=DEVICE)
            s["workspace"] = _gdn().recurrence.alloc_workspace(T, C, DEVICE)
        return s
    s["d_out"] = (torch.randn(*lead, C, generator=g, device=DEVICE) * 0.1).to(dtype)
    s["d_final"] = torch.randn(N, C, generator=g, device=DEVICE) * 0.1
    if own:
        for name in ("x", "a", "b", "A_log", "dt_bias") + (("state",) if case["state"] else ()):
            s[name] = s[name].detach().requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------
def _sigmoid(x):
    return 1.0 / (1.0 + torch.exp(-x))


def _softplus(x):
    return torch.clamp(x, min=0.0) + torch.log1p(torch.exp(-x.abs()))


def _gates(a, b, A_log, dt_bias):
    """log g, g, beta in fp32, and sigmoid(a + dt_bias)."""
    z = a.float() + dt_bias
    lg = -torch.exp(A_log) * _softplus(z)
    return lg, torch.exp(lg), _sigmoid(b.float()), z


def _scan(c, v, most):
    """y_t = c_t y_{t-1} + v_t along dim 0 by doubling (c, v are overwritten); no segment is longer than `most`."""
    s = 1
    while s < min(most, v.shape[0]):
        t = c[s:] * v[:-s]
        v[s:] += t
        t = c[s:] * c[:-s]
        c[s:] = t
        s *= 2
    return v


def _plain_forward(s, x, lg, g, beta):
    """All states [T, C] in fp32, and the one before each token."""
    cu, T = s["cu"], s["T"]
    C = x.shape[-1]
    starts = cu[:-1]
    h0 = s["state"] if s["state"] is not None else torch.zeros(s["N"], C, device=DEVICE)
    c, v = g.clone(), beta * x.float()
    v[starts] += g[starts] * h0
    c[starts] = 0.0
    h = _scan(c, v, max(s["lens"]))
    return h, h0


def _quantise(x):
    """The values that an 8-bit checkpoint of x [..., C] stands for (fp32)."""
    C = x.shape[-1]
    pad = -C % GROUP
    y = torch.nn.functional.pad(x.float(), (0, pad)).unflatten(-1, (-1, GROUP))
    m, e = torch.frexp(y.abs().amax(-1, keepdim=True))       # amax = m 2^e, m in [0.5, 1)
    e = torch.where(m <= 127.0 / 128.0, e - 7, e - 6)        # the smallest e with amax <= 127 2^e
    e = e.clamp(-126, TOP[x.dtype])
    q = torch.round(torch.ldexp(y, -e)).clamp(-127, 127)
    return torch.ldexp(q, e).flatten(-2)[..., :C]


def _plain_train(s, eight):
    case = s["case"]
    dtype, C, T = TYPES[case["type"]], case["channels"], s["T"]
    x, a, b = (s[n].reshape(T, C) for n in ("x", "a", "b"))
    d_out, cu = s["d_out"].reshape(T, C).float(), s["cu"]
    starts, ends = cu[:-1], cu[1:] - 1
    lg, g, beta, z = _gates(a, b, s["A_log"], s["dt_bias"])
    h, h0 = _plain_forward(s, x, lg, g, beta)
    out, final = h.to(dtype), h[ends].clone()
    before = torch.cat([torch.zeros(1, C, device=DEVICE), h[:-1]])
    before[starts] = h0
    if eight:
        x, a, b = _quantise(x), _quantise(a), _quantise(b)
        lg, g, beta, z = _gates(a, b, s["A_log"], s["dt_bias"])
        restart = torch.zeros(T, dtype=torch.bool, device=DEVICE)
        restart[::CHUNK] = True
        restart[starts] = True
        c, v = g.clone(), beta * x
        v[restart] += (g * before)[restart]
        c[restart] = 0.0
        inner = _scan(c, v, CHUNK)
        before = torch.where(restart[:, None], before, torch.cat([torch.zeros(1, C, device=DEVICE), inner[:-1]]))
        del c, v, inner
    # dh_t = d_out_t + g_{t+1} dh_{t+1}, from the last token back
    v = d_out.clone()
    v[ends] += s["d_final"]
    c = torch.cat([g[1:], torch.zeros(1, C, device=DEVICE)])
    c[ends] = 0.0
    dh = _scan(c.flip(0), v.flip(0), max(s["lens"])).flip(0)
    del c, v
    dlg = g * before * dh
    dx = (beta * dh).to(dtype)
    db = (x.float() * dh * beta * (1.0 - beta)).to(dtype)
    da = -torch.exp(s["A_log"]) * dlg * _sigmoid(z)
    dA_log, ddt_bias = (dlg * lg).sum(0), da.sum(0)
    shape = s["x"].shape
    got = {"out": out.view(shape), "final_state": final, "dx": dx.view(shape), "da": da.to(dtype).view(shape),
           "db": db.view(shape), "dA_log": dA_log, "ddt_bias": ddt_bias}
    if s["state"] is not None:
        got["d_state"] = g[starts] * dh[starts]
    return got


def _plain(s):
    case = s["case"]
    dtype, C = TYPES[case["type"]], case["channels"]
    if case["op"] == "pack":
        return [_quantise(t).to(t.dtype) for t in s["tensors"]]
    if case["op"] == "decode":
        x, a, b = (s[n].view(case["batch"], case["tokens"], C) for n in ("x", "a", "b"))
        lg, g, beta, z = _gates(a, b, s["A_log"], s["dt_bias"])
        u = beta * x.float()
        h = s["state"][s["slots"].long()] if case["pool"] else s["state"]
        steps = []
        for t in range(case["tokens"]):
            h = g[:, t] * h + u[:, t]
            steps.append(h)
        out = torch.stack(steps, 1).to(dtype).view(s["x"].shape)
        if case["pool"]:
            s["state"][s["slots"].long()] = h
            return out, s["state"]
        return out, h
    if case["op"] == "prefill":
        x, a, b = (s[n].reshape(s["T"], C) for n in ("x", "a", "b"))
        lg, g, beta, z = _gates(a, b, s["A_log"], s["dt_bias"])
        h, _ = _plain_forward(s, x, lg, g, beta)
        return h.to(dtype).view(s["x"].shape), h[s["cu"][1:] - 1]
    return _plain_train(s, case["op"] == "train8")


# ---------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------
def _own(s):
    case = s["case"]
    rec = _gdn().recurrence
    if case["op"] == "pack":
        ck = _gdn().checkpoint
        return ck.unpack(ck.pack(*s["tensors"]))
    if case["op"] == "decode":
        if case["pool"]:
            out = rec.decode_pool(s["x"], s["state"], s["slots"], s["A_log"], s["a"], s["dt_bias"], s["b"])
            return out, s["state"]
        return rec.decode(s["x"], s["state"], s["A_log"], s["a"], s["dt_bias"], s["b"])
    cu = None if s["dense"] else s["cu"]
    if case["op"] == "prefill":
        rec.run_into(s["x"], s["state"], s["A_log"], s["a"], s["dt_bias"], s["b"], cu, s["out"], s["final"],
                     s["workspace"])
        return s["out"], s["final"]
    out, final = rec.run_autograd(s["x"], s["state"], s["A_log"], s["a"], s["dt_bias"], s["b"], cu,
                                  checkpoint="int8" if case["op"] == "train8" else None)
    names = ["x", "a", "b", "A_log", "dt_bias"] + (["state"] if case["state"] else [])
    grads = torch.autograd.grad((out, final), [s[n] for n in names], (s["d_out"], s["d_final"]))
    got = {"out": out.detach(), "final_state": final.detach()}
    got.update({"d" + n if n != "state" else "d_state": v for n, v in zip(names, grads)})
    return got


def run(state):
    return _own(state) if state["own"] else _plain(state)


# ---------------------------------------------------------------------------
# the definition in 64 bits, token by token
# ---------------------------------------------------------------------------
def _exact_pack(t):
    y = t.double().cpu().numpy()
    flat = y.reshape(-1, y.shape[-1])
    got = np.empty_like(flat)
    for lo in range(0, flat.shape[1], GROUP):
        part = flat[:, lo:lo + GROUP]
        top = np.abs(part).max(1)
        e = np.full(top.shape, -126.0)
        some = top > 0
        e[some] = np.maximum(-126.0, np.ceil(np.log2(top[some] / 127.0)))
        e[top > 127.0 * 2.0 ** e] += 1           # log2 next to a whole number
        low = some & (top <= 127.0 * 2.0 ** (e - 1)) & (e > -126)
        e[low] -= 1
        unit = (2.0 ** np.minimum(e, TOP[t.dtype]))[:, None]
        got[:, lo:lo + GROUP] = np.clip(np.rint(part / unit), -127, 127) * unit
    return torch.from_numpy(got.reshape(y.shape))


def _sp64(z):
    return torch.logaddexp(z, torch.zeros_like(z))


def exact(case, seed):
    s = prepare(case, seed)
    C = case["channels"]
    if case["op"] == "pack":
        return [_exact_pack(t) for t in s["tensors"]]
    A, dt = s["A_log"].detach().double().exp(), s["dt_bias"].detach().double()
    x, a, b = (s[n].detach().double() for n in ("x", "a", "b"))
    if case["op"] == "decode":
        x, a, b = (t.view(case["batch"], case["tokens"], C) for t in (x, a, b))
        h = s["state"].double()
        if case["pool"]:
            pool, rows = h.clone(), s["slots"].long()
            h = h[rows]
        out = torch.empty_like(x)
        for t in range(case["tokens"]):
            h = torch.exp(-A * _sp64(a[:, t] + dt)) * h + torch.sigmoid(b[:, t]) * x[:, t]
            out[:, t] = h
        out = out.view(s["x"].shape)
        if case["pool"]:
            pool[rows] = h
            return out, pool
        return out, h
    T, N = s["T"], s["N"]
    x, a, b = (t.reshape(T, C) for t in (x, a, b))
    lens = np.array(s["lens"])
    order = np.argsort(-lens, kind="stable")             # the longest first: those still running are a prefix
    first = s["cu"][:-1][torch.from_numpy(order).to(DEVICE)]
    running = [int((lens > t).sum()) for t in range(int(lens.max()))]
    at = torch.from_numpy(order).to(DEVICE)
    h0 = s["state"].detach().double() if s["state"] is not None else torch.zeros(N, C, dtype=torch.float64, device=DEVICE)

    def forward(x, a, b, anchors=None):
        """h after each token; with `anchors` (states before each token) it starts anew from them at each chunk."""
        z = a + dt
        g = _sp64(z).mul_(-A).exp_()
        u = torch.sigmoid(b).mul_(x)
        if anchors is not None:
            whole = torch.empty_like(u)
            rows = torch.arange(0, T, CHUNK, device=DEVICE)
            cur = None
            for j in range(CHUNK):
                t = rows + j
                t = t[t < T]
                k = t.numel()
                new = is_start[t][:, None]
                prev = anchors[t] if j == 0 else torch.where(new, anchors[t], cur[:k])
                cur = g[t] * prev + u[t]
                whole[t] = cur
            return whole, g
        out = torch.empty_like(u)
        cur = h0[at].clone()
        for t, k in enumerate(running):
            rows = first[:k] + t
            cur[:k] = torch.addcmul(u[rows], g[rows], cur[:k])
            out[rows] = cur[:k]
        return out, g

    def shifted(h):
        prev = torch.empty_like(h)
        prev[1:] = h[:-1]
        prev[s["cu"][:-1]] = h0
        return prev

    h, g = forward(x, a, b)
    final = h[s["cu"][1:] - 1]
    shape = s["x"].shape
    if case["op"] == "prefill":
        return h.view(shape), final
    prev = shifted(h)
    is_start = torch.zeros(T, dtype=torch.bool, device=DEVICE)
    is_start[s["cu"][:-1]] = True
    if case["op"] == "train8":
        x, a, b = (_exact_pack(s[n].detach().reshape(T, C)).to(DEVICE) for n in ("x", "a", "b"))
        inner, g = forward(x, a, b, prev)
        keep = is_start.clone()
        keep[::CHUNK] = True
        nxt = torch.empty_like(inner)
        nxt[1:] = inner[:-1]
        nxt[keep] = prev[keep]
        prev = nxt
    d_out = s["d_out"].double().reshape(T, C)
    dh = torch.empty_like(d_out)
    d_state = torch.empty(N, C, dtype=torch.float64, device=DEVICE)
    carry = s["d_final"].double()[at].clone()
    last = first + torch.from_numpy(lens[order]).to(DEVICE) - 1
    for t, k in enumerate(running):                      # t tokens from the end
        rows = last[:k] - t
        cur = d_out[rows] + carry[:k]
        dh[rows] = cur
        carry[:k] = g[rows] * cur
    d_state[at] = carry
    beta = torch.sigmoid(b)
    z = a + dt
    dlg = g * prev * dh
    da = -A * dlg * torch.sigmoid(z)
    got = {"out": h.view(shape), "final_state": final, "dx": (beta * dh).view(shape), "da": da.view(shape),
           "db": (x * dh * beta * (1 - beta)).view(shape), "dA_log": (dlg * -A * _sp64(z)).sum(0), "ddt_bias": da.sum(0)}
    if s["state"] is not None:
        got["d_state"] = d_state
    return got


# ---------------------------------------------------------------------------
# the work that a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e, C = TYPES[case["type"]].itemsize, case["channels"]
    if case["op"] == "pack":
        n = case["rows"] * sum(map(int, case["heads"].split(","))) * C
        return {"bytes": 2 * n * e, "flops": 4 * n}
    if case["op"] == "decode":
        n, B = case["batch"] * case["tokens"] * C, case["batch"]
        return {"bytes": 4 * n * e + 8 * B * C + 8 * C, "flops": 12 * n}
    lens = _lengths(case, 0)
    n, N = sum(lens) * C, len(lens)
    states = 4 * N * C * (2 if case["state"] else 1)
    if case["op"] == "prefill":
        return {"bytes": 4 * n * e + states + 8 * C, "flops": 12 * n}
    # x, a, b and d_out in, out and three gradients out; the states' gradients besides
    return {"bytes": 8 * n * e + 2 * states + 16 * C, "flops": 40 * n}
