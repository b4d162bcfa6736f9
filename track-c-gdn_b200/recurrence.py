"""Channelwise gated linear recurrence: decode, prefill, backward.

The diagonal sibling of the GDN recurrence, with one fp32 state per channel
and the same gates, one per channel:

    g_t = exp(-exp(A_log) softplus(a_t + dt_bias)),  beta_t = sigmoid(b_t)
    h_t = g_t h_{t-1} + beta_t x_t,  out_t = h_t

x, a, b are bf16, fp16 or fp32 (one type for the three; outputs and gradients
have it too), A_log and dt_bias [D] and states [N, D] fp32.  Sequences are
packed ([T, D] with `cu_seqlens` [N+1] int64) or dense ([N, S, D] without).
The channels of a token must lie next to one another; tokens may be apart, so
x, a and b may be slices of one projection's output (any other layout is
copied first).  Everything is computed and carried in fp32, and a result is
rounded once, when it is stored.  Behind an infinite state the outputs are not
finite, infinite or NaN (products of gates may underflow to 0).

Nothing here synchronises the host.  cu_seqlens and slots are checked on the
device: bad values are reported by `_native.read_device_status` (1 and 3) and
the call writes nothing.  cu_seqlens[-1] may be less than T; the rows behind
the last sequence are zero in what `run`, `run_pool`, `backward` and
`run_autograd` return, and left as they were by the `_into` forms.  A call may
be captured into a CUDA graph; calls that overlap in time, among them replays
of two graphs, need a workspace each (the value-returning forms allocate their
own).  No counterpart in the reference.
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native

CHUNK = 64               # rows between two saved states
DECODE_MAX_TOKENS = 64

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _copied(t: torch.Tensor, stream):
    """A contiguous copy, made on the current stream -- which a call on another
    stream would not wait for."""
    if stream is not None:
        raise ValueError("with `stream` the inputs must be laid out as the kernels read them "
                         "(channels side by side, one distance between tokens)")
    return t.detach().contiguous()


def _rows(t: torch.Tensor, stream=None):
    """`t` as rows of channels: (tensor that owns them, elements between rows)."""
    strides, shape = t.stride(), t.shape
    if strides[-1] != 1 and shape[-1] != 1:
        t = _copied(t, stream)
        strides = t.stride()
    if len(strides) == 2:
        return t, strides[0]
    if shape[0] != 1 and shape[1] != 1 and strides[0] != shape[1] * strides[1]:
        t = _copied(t, stream)
        strides = t.stride()
    return t, (strides[0] if shape[1] == 1 else strides[1])


def _vector(t: torch.Tensor, stream):
    return t if t.is_contiguous() else _copied(t, stream)


def _check_inputs(x, a, b, A_log, dt_bias):
    if x.dtype not in _TYPES:
        raise TypeError(f"the recurrence expects bf16, fp16 or fp32 x, got {x.dtype}")
    if a.dtype != x.dtype or b.dtype != x.dtype:
        raise TypeError(f"a ({a.dtype}) and b ({b.dtype}) must have x's type {x.dtype}")
    if A_log.dtype != torch.float32 or dt_bias.dtype != torch.float32:
        raise TypeError("A_log and dt_bias must be fp32")
    if not x.is_cuda:
        raise ValueError(f"the recurrence expects CUDA tensors (x is on {x.device})")
    for name, t in (("a", a), ("b", b), ("A_log", A_log), ("dt_bias", dt_bias)):
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    assert x.dim() in (2, 3) and x.shape[-1] >= 1, "x must be [T, D] or [N, S, D]"
    assert a.shape == x.shape and b.shape == x.shape, "a and b must have x's shape"
    D = x.shape[-1]
    assert A_log.shape == (D,) and dt_bias.shape == (D,), "A_log and dt_bias must be [D]"
    return D


def _check_states(name, t, rows, D, device):
    assert t.dtype == torch.float32 and t.shape == (rows, D), f"{name} must be [{rows}, {D}] fp32"
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, x on {device}")


def _sequences(x, cu_seqlens):
    """(T, N, pointer of cu_seqlens)."""
    if cu_seqlens is None:
        if x.dim() == 2:
            return x.shape[0], 1, None
        return x.shape[0] * x.shape[1], x.shape[0], None
    assert x.dim() == 2, "with cu_seqlens x must be packed, [T, D]"
    assert cu_seqlens.dtype == torch.int64 and cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 1
    assert cu_seqlens.is_contiguous(), "cu_seqlens must be contiguous"
    if cu_seqlens.device != x.device:
        raise ValueError(f"cu_seqlens is on {cu_seqlens.device}, x on {x.device}")
    return x.shape[0], cu_seqlens.numel() - 1, cu_seqlens.data_ptr()


def _check_slots(slots, count, pool, D, device):
    assert pool.dim() == 2 and pool.shape[1] == D and pool.dtype == torch.float32, "the pool must be [P, D] fp32"
    assert pool.is_contiguous(), "the pool must be contiguous"
    assert slots.dtype == torch.int32 and slots.numel() == count and slots.is_contiguous(), \
        f"slots must be {count} contiguous int32"
    if pool.device != device or slots.device != device:
        raise ValueError(f"the pool ({pool.device}) and slots ({slots.device}) must be on {device}")


_current_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _call(fn, device, args, stream):
    """Calls the library's `fn` with `device` current, on `stream` or the
    device's current stream."""
    index = device.index
    if stream is None:
        stream = _current_stream(index)
    if index == _current_device():
        st = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            st = fn(*args, stream)
    if st:
        _native.check(st, fn.__name__)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------
def decode_into(x, state, A_log, a, dt_bias, b, out, new_state, slots: Optional[torch.Tensor] = None,
                intermediate: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> None:
    """One token ([B, D]) or up to 64 in order ([B, T, D]) for each request.
    Writes `out` (x's shape, contiguous) and `new_state` [B, D], which may be
    `state` ([B, D], None: zeros).  With `slots` ([B] int32, distinct) both are
    one pool [P, D], updated in place; a request whose slot is outside the pool
    is skipped (device status 3).  `intermediate` [B, T, D] fp32 receives the
    state after each token.  `out` may be x, a or b itself, if that is
    contiguous; no output may share memory with an input otherwise."""
    D = _check_inputs(x, a, b, A_log, dt_bias)
    B, T = x.shape[0], (x.shape[1] if x.dim() == 3 else 1)
    assert 1 <= T <= DECODE_MAX_TOKENS, f"1 <= T <= {DECODE_MAX_TOKENS}"
    device = x.device
    if slots is not None:
        assert state is not None and state.data_ptr() == new_state.data_ptr(), "a pool is updated in place"
        _check_slots(slots, B, state, D, device)
    else:
        if state is not None:
            _check_states("state", state, B, D, device)
            assert state.is_contiguous(), "state must be contiguous"
        _check_states("new_state", new_state, B, D, device)
    assert out.shape == x.shape and out.dtype == x.dtype and out.is_contiguous() and out.device == device
    assert new_state.is_contiguous()
    if intermediate is not None:
        assert intermediate.shape == (B, T, D) and intermediate.dtype == torch.float32
        assert intermediate.is_contiguous() and intermediate.device == device
    x, xs = _rows(x, stream)
    a, as_ = _rows(a, stream)
    b, bs = _rows(b, stream)
    A_log, dt_bias = _vector(A_log, stream), _vector(dt_bias, stream)
    _call(_native.lib.gdn_recurrence_decode, device,
          (_TYPES[x.dtype], x.data_ptr(), xs, a.data_ptr(), as_, b.data_ptr(), bs, A_log.data_ptr(),
           dt_bias.data_ptr(), _ptr(state), _ptr(slots), 0 if slots is None else state.shape[0], B, T, D,
           out.data_ptr(), new_state.data_ptr(), _ptr(intermediate)), stream)


def decode(x, state, A_log, a, dt_bias, b, return_intermediate: bool = False):
    """Decode with a fresh new state: x, a, b [B, D] or [B, T, D], state [B, D]
    fp32 or None.  Returns (out, new_state), and with return_intermediate the
    states after each token [B, T, D] fp32 too."""
    out = x.new_empty(x.shape)
    new_state = (torch.empty(x.shape[0], x.shape[-1], dtype=torch.float32, device=x.device) if state is None
                 else state.new_empty(state.shape))
    inter = None
    if return_intermediate:
        T = x.shape[1] if x.dim() == 3 else 1
        inter = torch.empty(x.shape[0], T, x.shape[-1], dtype=torch.float32, device=x.device)
    decode_into(x, None if state is None else state.contiguous(), A_log, a, dt_bias, b, out, new_state,
                intermediate=inter)
    return (out, new_state, inter) if return_intermediate else (out, new_state)


def decode_inplace(x, state, A_log, a, dt_bias, b):
    """Decode with `state` [B, D] updated in place.  Returns out."""
    out = x.new_empty(x.shape)
    decode_into(x, state, A_log, a, dt_bias, b, out, state)
    return out


def decode_pool(x, state_pool, slots, A_log, a, dt_bias, b):
    """Decode with request i's state in state_pool[slots[i]] ([P, D] fp32,
    updated in place; slots [B] int32, distinct).  Returns out."""
    out = x.new_empty(x.shape)
    decode_into(x, state_pool, A_log, a, dt_bias, b, out, state_pool, slots=slots)
    return out


# ---------------------------------------------------------------------------
# prefill
# ---------------------------------------------------------------------------
@lru_cache(maxsize=256)
def workspace_bytes(total_tokens: int, channels: int) -> int:
    return int(_native.lib.gdn_recurrence_workspace_bytes(total_tokens, channels))


def alloc_workspace(total_tokens: int, channels: int, device) -> torch.Tensor:
    """A workspace for `run_into` (1 KiB of slack for the 1024-byte alignment).
    Calls that overlap in time need one each."""
    return torch.empty(workspace_bytes(total_tokens, channels) + 1024, dtype=torch.uint8, device=device)


def _prefill(x, state, A_log, a, dt_bias, b, cu_seqlens, out, final_state, workspace, slots=None, carries=None,
             packed=None, zero_behind=False, stream=None):
    D = _check_inputs(x, a, b, A_log, dt_bias)
    T, N, cu = _sequences(x, cu_seqlens)
    device = x.device
    if slots is not None:
        _check_slots(slots, N, state, D, device)
    else:
        if state is not None:
            _check_states("state", state, N, D, device)
            assert state.is_contiguous(), "state must be contiguous"
        _check_states("final_state", final_state, N, D, device)
        assert final_state.is_contiguous(), "final_state must be contiguous"
    assert out.shape == x.shape and out.dtype == x.dtype and out.is_contiguous() and out.device == device
    _launch_prefill(x, state, A_log, a, dt_bias, b, (T, N, cu), out, final_state, workspace, slots, carries, packed,
                    zero_behind, stream)


def _launch_prefill(x, state, A_log, a, dt_bias, b, seqs, out, final_state, workspace, slots, carries, packed,
                    zero_behind, stream):
    T, N, cu = seqs
    wptr, wbytes = _native.aligned_workspace(workspace, x.device)
    x, xs = _rows(x, stream)
    a, as_ = _rows(a, stream)
    b, bs = _rows(b, stream)
    A_log, dt_bias = _vector(A_log, stream), _vector(dt_bias, stream)
    _call(_native.lib.gdn_recurrence_prefill, x.device,
          (_TYPES[x.dtype], x.data_ptr(), xs, a.data_ptr(), as_, b.data_ptr(), bs, A_log.data_ptr(),
           dt_bias.data_ptr(), _ptr(state), _ptr(slots), 0 if slots is None else state.shape[0], cu, N, T,
           x.shape[-1], int(zero_behind), out.data_ptr(), final_state.data_ptr(), _ptr(carries), _ptr(packed), wptr,
           wbytes), stream)


def run_into(x, state, A_log, a, dt_bias, b, cu_seqlens, out, final_state, workspace: torch.Tensor,
             stream: Optional[int] = None) -> None:
    """Destination-passing prefill: writes `out` (x's shape) and `final_state`
    [N, D] fp32 (may be `state`).  Rows behind the last sequence are left as
    they were."""
    _prefill(x, state, A_log, a, dt_bias, b, cu_seqlens, out, final_state, workspace, stream=stream)


def run(x, state, A_log, a, dt_bias, b, cu_seqlens: Optional[torch.Tensor] = None):
    """Prefill of packed (x [T, D], cu_seqlens [N+1] int64) or dense sequences
    (x [N, S, D], or one sequence [S, D]).  state [N, D] fp32 or None.  Returns
    (out, final_state [N, D] fp32)."""
    T, N, _ = _sequences(x, cu_seqlens)
    D = x.shape[-1]
    out = x.new_empty(x.shape)
    final_state = torch.empty(N, D, dtype=torch.float32, device=x.device)
    _prefill(x, None if state is None else state.contiguous(), A_log, a, dt_bias, b, cu_seqlens, out, final_state,
             alloc_workspace(T, D, x.device), zero_behind=True)
    return out, final_state


def run_pool_into(x, state_pool, slots, A_log, a, dt_bias, b, cu_seqlens, out, workspace: torch.Tensor,
                  stream: Optional[int] = None) -> None:
    """Destination-passing prefill against a state pool: sequence n starts from
    state_pool[slots[n]] ([P, D] fp32) and leaves its final state there."""
    _prefill(x, state_pool, A_log, a, dt_bias, b, cu_seqlens, out, state_pool, workspace, slots=slots,
             stream=stream)


def run_pool(x, state_pool, slots, A_log, a, dt_bias, b, cu_seqlens: Optional[torch.Tensor] = None):
    """`run` with the states in a pool ([P, D] fp32, updated in place at
    slots [N] int32, distinct).  Returns out."""
    T, _, _ = _sequences(x, cu_seqlens)
    out = x.new_empty(x.shape)
    _prefill(x, state_pool, A_log, a, dt_bias, b, cu_seqlens, out, state_pool,
             alloc_workspace(T, x.shape[-1], x.device), slots=slots, zero_behind=True)
    return out


# ---------------------------------------------------------------------------
# backward
# ---------------------------------------------------------------------------
@lru_cache(maxsize=256)
def backward_workspace_bytes(total_tokens: int, channels: int) -> int:
    return int(_native.lib.gdn_recurrence_backward_workspace_bytes(total_tokens, channels))


def alloc_backward_workspace(total_tokens: int, channels: int, device) -> torch.Tensor:
    """A workspace for `backward_into` (1 KiB of slack for the alignment)."""
    return torch.empty(backward_workspace_bytes(total_tokens, channels) + 1024, dtype=torch.uint8, device=device)


def _backward(x, state, A_log, a, dt_bias, b, cu_seqlens, d_out, d_final_state, dx, da, db, dA_log, ddt_bias,
              d_state, workspace, carries=None, packed=None, zero_behind=False, stream=None):
    """x, a, b may be None with `packed`; shapes and type then are d_out's."""
    device, dtype, D = d_out.device, d_out.dtype, d_out.shape[-1]
    T, N, cu = _sequences(d_out, cu_seqlens)
    for t in (dx, da, db):
        assert t.shape == d_out.shape and t.dtype == dtype and t.is_contiguous() and t.device == device
    for t in (dA_log, ddt_bias):
        assert t.shape == (D,) and t.dtype == torch.float32 and t.is_contiguous() and t.device == device
    for name, t in (("state", state), ("d_final_state", d_final_state), ("d_state", d_state)):
        if t is not None:
            _check_states(name, t, N, D, device)
            assert t.is_contiguous(), f"{name} must be contiguous"
    if packed is None:
        _check_inputs(x, a, b, A_log, dt_bias)
        assert x.shape == d_out.shape and x.dtype == dtype and x.device == device, "d_out must be like x"
    _launch_backward(x, state, A_log, a, dt_bias, b, (T, N, cu), d_out, d_final_state,
                     (dx, da, db, dA_log, ddt_bias, d_state), workspace, carries, packed, zero_behind, stream)


def _launch_backward(x, state, A_log, a, dt_bias, b, seqs, d_out, d_final_state, grads, workspace, carries, packed,
                     zero_behind, stream):
    T, N, cu = seqs
    wptr, wbytes = _native.aligned_workspace(workspace, d_out.device)
    xs = as_ = bs = 0
    if packed is None:
        x, xs = _rows(x, stream)
        a, as_ = _rows(a, stream)
        b, bs = _rows(b, stream)
    d_out, ds = _rows(d_out, stream)
    A_log, dt_bias = _vector(A_log, stream), _vector(dt_bias, stream)
    dx, da, db, dA_log, ddt_bias, d_state = grads
    _call(_native.lib.gdn_recurrence_backward, d_out.device,
          (_TYPES[d_out.dtype], _ptr(x), xs, _ptr(a), as_, _ptr(b), bs, _ptr(packed), A_log.data_ptr(),
           dt_bias.data_ptr(), _ptr(state), cu, N, T, d_out.shape[-1], int(zero_behind), d_out.data_ptr(), ds,
           _ptr(d_final_state), _ptr(carries), dx.data_ptr(), da.data_ptr(), db.data_ptr(), dA_log.data_ptr(),
           ddt_bias.data_ptr(), _ptr(d_state), wptr, wbytes), stream)


def backward_into(x, state, A_log, a, dt_bias, b, cu_seqlens, d_out, d_final_state, dx, da, db, dA_log, ddt_bias,
                  d_state, workspace: torch.Tensor, stream: Optional[int] = None) -> None:
    """Destination-passing backward: gradients dx, da, db (x's shape and type),
    dA_log, ddt_bias [D] fp32 and (unless None) d_state [N, D] fp32 of
    `run(x, state, A_log, a, dt_bias, b, cu_seqlens)` from d_out (like x) and
    d_final_state [N, D] fp32 (None: zero).  Runs the recurrence once more to
    find the chunks' states.  Rows behind the last sequence are left as they
    were."""
    _backward(x, state, A_log, a, dt_bias, b, cu_seqlens, d_out, d_final_state, dx, da, db, dA_log, ddt_bias,
              d_state, workspace, stream=stream)


_NAMES = ("dx", "da", "db", "dA_log", "ddt_bias", "d_state")


def _gradients(like, D, N, need_d_state):
    shape, params = like.shape, torch.empty(D, dtype=torch.float32, device=like.device)
    return (like.new_empty(shape), like.new_empty(shape), like.new_empty(shape), params, params.new_empty(D),
            params.new_empty((N, D)) if need_d_state else None)


@torch.no_grad()
def backward(x, state, A_log, a, dt_bias, b, cu_seqlens, d_out, d_final_state=None, need_d_state: bool = True):
    """Gradients of `run(x, state, A_log, a, dt_bias, b, cu_seqlens)`.  Returns
    a dict: dx, da, db (x's shape and type), dA_log, ddt_bias [D] fp32, d_state
    [N, D] fp32 (None unless need_d_state)."""
    T, N, _ = _sequences(x, cu_seqlens)
    D = x.shape[-1]
    g = _gradients(x, D, N, need_d_state)
    _backward(x, None if state is None else state.contiguous(), A_log, a, dt_bias, b, cu_seqlens, d_out.to(x.dtype),
              None if d_final_state is None else d_final_state.float().contiguous(), *g,
              alloc_backward_workspace(T, D, x.device), zero_behind=True)
    return dict(zip(_NAMES, g))


@lru_cache(maxsize=256)
def _saved_bytes(total_tokens: int, channels: int):
    lib = _native.lib
    return (int(lib.gdn_recurrence_carry_bytes(total_tokens, channels)),
            int(lib.gdn_recurrence_packed_bytes(total_tokens, channels)))


class _RecurrenceFunction(torch.autograd.Function):
    """run(...) with gradients.  The forward keeps the state before every 64th
    row (1/32 of x's bytes for a 2-byte type), and x, a, b themselves or their
    8-bit form."""

    @staticmethod
    def forward(ctx, x, state, A_log, a, dt_bias, b, cu_seqlens, checkpoint):
        D = _check_inputs(x, a, b, A_log, dt_bias)
        seqs = T, N, _ = _sequences(x, cu_seqlens)
        dev = x.device
        if state is not None:
            _check_states("state", state, N, D, dev)
            state = state.contiguous()
        out = x.new_empty(x.shape)
        final_state = torch.empty(N, D, dtype=torch.float32, device=dev)
        carry_bytes, packed_bytes = _saved_bytes(T, D)
        carries = torch.empty(carry_bytes, dtype=torch.uint8, device=dev)
        packed = None
        if checkpoint is not None:
            packed = torch.empty(packed_bytes, dtype=torch.uint8, device=dev)
        _launch_prefill(x, state, A_log, a, dt_bias, b, seqs, out, final_state, alloc_workspace(T, D, dev), None,
                        carries, packed, True, None)
        if packed is None:
            ctx.save_for_backward(x, a, b, None, state, A_log, dt_bias, cu_seqlens, carries)
        else:
            ctx.save_for_backward(None, None, None, packed, state, A_log, dt_bias, cu_seqlens, carries)
        ctx.like = (x.shape, x.dtype, dev, T, N)
        ctx.set_materialize_grads(False)
        return out, final_state

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_final):
        x, a, b, packed, state, A_log, dt_bias, cu_seqlens, carries = ctx.saved_tensors
        shape, dtype, dev, T, N = ctx.like
        if d_out is None:
            d_out = torch.zeros(shape, dtype=dtype, device=dev)
        D = shape[-1]
        g = _gradients(d_out, D, N, state is not None and ctx.needs_input_grad[1])
        _launch_backward(x, state, A_log, a, dt_bias, b, (T, N, _ptr(cu_seqlens)), d_out,
                         None if d_final is None else d_final.contiguous(), g, alloc_backward_workspace(T, D, dev),
                         carries, packed, True, None)
        dx, da, db, dA_log, ddt_bias, d_state = g
        return dx, d_state, dA_log, da, ddt_bias, db, None, None


def run_autograd(x, state, A_log, a, dt_bias, b, cu_seqlens: Optional[torch.Tensor] = None,
                 checkpoint: Optional[str] = None):
    """`run` with gradients for torch.autograd, in x, state, A_log, a, dt_bias
    and b (first order only).

    checkpoint="int8" keeps x, a and b until the backward in 8 bits (the format
    of `checkpoint.pack`, written and read by the recurrence's own kernels)
    instead of as they are: half the bytes for 2-byte types.  The outputs do
    not change; the gradients are those at the 8-bit values, with the states
    before the tokens restarted from exact ones at every 64th row."""
    if checkpoint not in (None, "int8"):
        raise ValueError(f"checkpoint must be None or 'int8', got {checkpoint!r}")
    return _RecurrenceFunction.apply(x, state, A_log, a, dt_bias, b, cu_seqlens, checkpoint)
