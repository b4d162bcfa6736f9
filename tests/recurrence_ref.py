"""The channelwise gated linear recurrence and the 8-bit checkpoint format from
their definitions in float64 on the CPU, token by token, with bounds on what
fp32 evaluation may be off by.

A bound counts the roundings of one token's work in units of u = 2^-24 and
carries them through the recurrence on absolute values (so any order of
evaluation, also of composed affine maps, is covered):
  exp by one base-2 exponential: its argument is rounded (a relative error of
    2 u in the argument is |argument| 2 u in the result) and it is accurate to
    2^-22 = 4 u
  w = (a + dt_bias) log2(e) as one fused a log2(e) + fl(dt_bias log2(e)): off by
    log2(e) u (|a| + 2 |dt_bias| + |z|), which moves softplus by at most its
    slope times that, and the slope is at most softplus itself
  softplus: besides, the exponential 4 u, the logarithm's polynomial 3 u, sum 1 u:
    (|a| + 2 |dt_bias| + |z| + 8) u
  lg = -exp(A_log) softplus: exp(A_log) 4 u and two products: 15 for the 8
  g = exp(lg): |lg| times lg's and 4 u
  sigmoid: (2 |b| + 8) u; u_t = sigmoid(b) x one more
  a state: the product and sum of its update, and as much again where maps
    are composed: 3 u of the sum's absolute parts
"""
from __future__ import annotations

import torch

U = 2.0 ** -24
CHUNK = 64
GROUP = 128
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
TOP_EXPONENT = {torch.bfloat16: 121, torch.float16: 9, torch.float32: 121}


def softplus(z):
    return torch.logaddexp(z, torch.zeros_like(z))


class Gates:
    """Per token and channel in float64: g, beta, u and their relative errors."""

    def __init__(self, x, a, b, A_log, dt_bias):
        x, a, b = x.double(), a.double(), b.double()
        self.x, self.A = x, A_log.double().exp()
        self.z = a + dt_bias.double()
        self.sp = softplus(self.z)
        self.lg = -self.A * self.sp
        self.g = self.lg.exp()
        self.beta = torch.sigmoid(b)
        self.u = self.beta * x
        self.moved = a.abs() + 2 * dt_bias.double().abs() + self.z.abs()
        self.rel_lg = (self.moved + 15) * U
        self.rel_g = self.lg.abs() * self.rel_lg + 4 * U
        self.rel_beta = (2 * b.abs() + 8) * U
        self.rel_u = self.rel_beta + U


def ranges(cu):
    return [(int(s), int(e)) for s, e in zip(cu[:-1], cu[1:])]


def _states(k: Gates, cu, first, first_err):
    """h after each token, bounds, and both before each token; `first` [N, D]."""
    h, err, prev, prev_err = (torch.zeros_like(k.u) for _ in range(4))
    last, last_err = first.clone(), first_err.clone()
    for n, (s, e) in enumerate(ranges(cu)):
        v, r, mag = first[n], first_err[n], first[n].abs()
        for t in range(s, e):
            prev[t], prev_err[t] = v, r
            r = k.g[t] * (r + mag * (k.rel_g[t] + 2 * U)) + k.u[t].abs() * k.rel_u[t]
            v = k.g[t] * v + k.u[t]
            mag = k.g[t] * mag + k.u[t].abs()
            r = r + 3 * U * mag
            h[t], err[t] = v, r
        last[n], last_err[n] = v, r
    return h, err, prev, prev_err, last, last_err


def forward(x, state, A_log, a, dt_bias, b, cu):
    """dict of (value, bound): out [T, D] (before rounding), final_state [N, D]."""
    k = Gates(x, a, b, A_log, dt_bias)
    N, D = len(cu) - 1, x.shape[1]
    h0 = torch.zeros(N, D, dtype=torch.float64) if state is None else state.double()
    h, err, _, _, last, last_err = _states(k, cu, h0, torch.zeros_like(h0))
    return {"out": (h, err), "final_state": (last, last_err)}


def quantise(x):
    """The values that the 8-bit form of x [..., C] stands for, from the
    definition (float64, exact)."""
    y = x.double()
    got = torch.empty_like(y)
    top_e = TOP_EXPONENT[x.dtype]
    for lo in range(0, y.shape[-1], GROUP):
        part = y[..., lo:lo + GROUP]
        top = part.abs().amax(-1, keepdim=True)
        e = torch.full_like(top, -126.0)
        fine = torch.isfinite(top)
        for cand in range(-126, top_e):      # the smallest e with max <= 127 2^e, as far as top_e
            e = torch.where(fine & (top > 127.0 * 2.0 ** cand), torch.full_like(e, cand + 1.0), e)
        unit = torch.pow(torch.full_like(e, 2.0), e)
        q = torch.round(part / unit).clamp(-127, 127)
        got[..., lo:lo + GROUP] = torch.where(fine, q * unit, torch.full_like(part, float("nan")))
    return got


def backward(x, state, A_log, a, dt_bias, b, cu, d_out, d_final, eight=False):
    """dict of (value, bound) of the gradients, before they are rounded."""
    T, D = x.shape
    N = len(cu) - 1
    k = Gates(x, a, b, A_log, dt_bias)
    h0 = torch.zeros(N, D, dtype=torch.float64) if state is None else state.double()
    _, _, prev, prev_err, _, _ = _states(k, cu, h0, torch.zeros_like(h0))
    if eight:
        x, a, b = quantise(x), quantise(a), quantise(b)
        k = Gates(x, a, b, A_log, dt_bias)
        # states before the tokens, anew from the exact ones at each 64th row
        first, first_err = prev.clone(), prev_err.clone()
        for s, e in ranges(cu):
            for t in range(s, e):
                if t == s or t % CHUNK == 0:
                    v, r, mag = first[t], first_err[t], first[t].abs()
                prev[t], prev_err[t] = v, r
                r = k.g[t] * (r + mag * (k.rel_g[t] + 2 * U)) + k.u[t].abs() * k.rel_u[t]
                v = k.g[t] * v + k.u[t]
                mag = k.g[t] * mag + k.u[t].abs()
                r = r + 3 * U * mag
    do = d_out.double()
    df = torch.zeros(N, D, dtype=torch.float64) if d_final is None else d_final.double()
    dh, dh_err = torch.zeros_like(do), torch.zeros_like(do)
    d_state, d_state_err = df.clone(), torch.zeros_like(df)
    for n, (s, e) in enumerate(ranges(cu)):
        R, r, mag = df[n], torch.zeros(D, dtype=torch.float64), df[n].abs()
        for t in range(e - 1, s - 1, -1):
            v, mag = do[t] + R, do[t].abs() + mag
            dh[t], dh_err[t] = v, r + U * mag
            r = k.g[t] * (r + mag * (k.rel_g[t] + 4 * U))
            R, mag = k.g[t] * v, k.g[t] * mag
        d_state[n], d_state_err[n] = R, r + 2 * U * mag
    sig = torch.sigmoid(k.z)
    # sigmoid(z) = exp(z - softplus(z)) by one exponential: w and softplus are off
    # as above, their difference is rounded, 4 u for the exponential
    rel_sig = (2 * k.moved + 3 * k.sp + 16) * U + k.sp * (k.moved + 8) * U
    slope = k.beta * (1 - k.beta)
    dx = k.beta * dh
    dx_err = dx.abs() * (k.rel_beta + U) + k.beta * dh_err
    db = k.x * dh * slope
    # beta - beta^2 in one rounding from the rounded beta: its error is beta's
    # times |1 - 2 beta| <= 1, also where 1 - beta is small
    db_err = (k.x * dh).abs() * k.beta * k.rel_beta + db.abs() * 4 * U + (k.x * slope).abs() * dh_err
    dlg = k.g * prev * dh
    dlg_err = dlg.abs() * (k.rel_g + 3 * U) + k.g * (dh.abs() * prev_err + prev.abs() * dh_err)
    da = -k.A * dlg * sig
    da_err = da.abs() * (rel_sig + 9 * U) + (k.A * sig) * dlg_err
    terms = dlg * k.lg
    terms_err = terms.abs() * (k.rel_lg + 3 * U) + k.lg.abs() * dlg_err
    chunks = max(1, -(-T // CHUNK))
    adds = (8 + 8 + -(-chunks // 32) + 32) * U      # a lane's tokens, the warps, the chunks of a thread, the threads
    return {"dx": (dx, dx_err), "da": (da, da_err), "db": (db, db_err),
            "dA_log": (terms.sum(0), terms_err.sum(0) + adds * terms.abs().sum(0)),
            "ddt_bias": (da.sum(0), da_err.sum(0) + adds * da.abs().sum(0)),
            "d_state": (d_state, d_state_err)}


def assert_close(got, want, what, dtype=None):
    """|got - value| <= bound + half a step of `dtype` (fp32 results: none)."""
    value, bound = want
    got = got.double().cpu().reshape(value.shape)
    tol = bound + 1e-30
    if dtype is not None and dtype != torch.float32:
        tol = tol + HALF_STEP[dtype] * (value.abs() + bound) + TINY[dtype]
    bad = ~((got - value).abs() <= tol)
    if bool(bad.any()):
        i = int(torch.nonzero(bad.flatten())[0])
        ratio = ((got - value).abs() / tol).max().item()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {got.flatten()[i].item()!r} "
                             f"for {value.flatten()[i].item()!r}, largest error / bound {ratio:.3g}")
