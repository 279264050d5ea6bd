"""The gated delta rule on the B200: whole sequences, and one token at a time.

A value head carries a K x V matrix S instead of the scans' one number for
each channel, and each token replaces what the state holds for its key:

    S_t = a_t S_{t-1} + k_t u_t^T,   a_t = exp(log_decay_t)
    u_t = beta_t (v_t - (a_t S_{t-1})^T k_t)
    o_t = scale S_t^T q_t

gated_delta_scan takes sequences (training, prompts), gated_delta_step one
token for each row on states in a pool (serving).  The reference has no
matrix-state recurrence; its selective scan
(rqf_models/ops/selective_scan.py:107-170) is the nearest thing to it.  As in
ops.py there is no CPU fallback: other tensors raise.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _abi, _timing
from .ops import _done, _nbytes, _require_cuda, _scratch

__all__ = ["gated_delta_scan", "gated_delta_step"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_KEY_DIM = 128


def _check(q, k, v, log_decay, beta, lead: int) -> None:
    """Shapes and types of one call; `lead` axes (batch, or batch and time) before the heads."""
    names = ("q", "k", "v", "log_decay", "beta")
    for name, t, extra in zip(names, (q, k, v, log_decay, beta), (2, 2, 2, 1, 1)):
        if t.dim() != lead + extra:
            raise ValueError(f"{name} must have {lead + extra} axes, got shape {tuple(t.shape)}")
    if v.dtype not in _DTYPES or q.dtype != v.dtype or k.dtype != v.dtype:
        raise ValueError("q, k and v must all be float32, bfloat16 or float16, got "
                         f"{q.dtype}, {k.dtype}, {v.dtype}")
    for name, t in (("log_decay", log_decay), ("beta", beta)):
        if not t.dtype.is_floating_point:
            raise ValueError(f"{name} must be floating point, got {t.dtype}")
    if k.shape != q.shape:
        raise ValueError(f"q and k must have one shape, got {tuple(q.shape)} and {tuple(k.shape)}")
    if v.shape[:lead] != q.shape[:lead]:
        raise ValueError(f"q and v do not match: {tuple(q.shape)} and {tuple(v.shape)}")
    for name, t in (("log_decay", log_decay), ("beta", beta)):
        if t.shape != v.shape[:-1]:
            raise ValueError(f"{name} must have shape {tuple(v.shape[:-1])}, got {tuple(t.shape)}")
    hk, dk = q.shape[-2:]
    hv, dv = v.shape[-2:]
    if hk == 0 or hv == 0 or hv % hk:
        raise ValueError(f"{hv} value heads cannot share {hk} key heads")
    if dk == 0 or dv == 0 or dk % 8 or dv % 8 or dk > MAX_KEY_DIM:
        raise ValueError("head sizes must be multiples of 8 and the keys' at most "
                         f"{MAX_KEY_DIM}, got {dk} and {dv}")


def _check_state(state, shape, name) -> None:
    if state.dtype != torch.float32 or tuple(state.shape) != tuple(shape):
        raise ValueError(f"{name} must be float32 {tuple(shape)}, got {state.dtype} {tuple(state.shape)}")


def _dense16(t: torch.Tensor) -> torch.Tensor:
    """t itself where its last axis is dense and rows start on 16 bytes, else a copy."""
    if t.numel() == 0:
        return t
    per = 16 // t.element_size()
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % per == 0 for s in t.stride()[:-1]):
        return t
    return t.contiguous() if t.data_ptr() % 16 == 0 or not t.is_contiguous() else t.clone()


def _problem(q, k, v, log_decay, beta, lengths, scale) -> "_abi.DeltaProblem":
    """The C description of a call on (batch, time, heads, ...) tensors, or (batch, heads, ...)."""
    p = _abi.DeltaProblem()
    steps = v.dim() == 4
    p.batch, p.time = v.shape[0], v.shape[1] if steps else 1
    p.key_heads, p.key_dim = q.shape[-2:]
    p.value_heads, p.value_dim = v.shape[-2:]
    for name, t in (("q", q), ("k", k), ("v", v), ("g", log_decay), ("beta", beta)):
        s = t.stride()
        getattr(p, f"{name}_stride")[:] = (s[0], s[1], s[2]) if steps else (s[0], 0, s[1])
    p.lengths = None if lengths is None else lengths.data_ptr()
    p.dtype = _DTYPES[v.dtype]
    p.scale = scale
    return p


class _GatedDeltaScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, beta, initial_state, lengths, scale, save):
        dev = _require_cuda(q, k, v, log_decay, beta, initial_state, lengths)
        q, k, v = (_dense16(t.detach()) for t in (q, k, v))
        g, b = log_decay.detach(), beta.detach()
        s0 = None if initial_state is None else initial_state.detach().contiguous()
        B, T, Hv, V = v.shape
        K = q.shape[-1]
        o = torch.empty((B, T, Hv, V), dtype=v.dtype, device=dev)
        last = torch.empty((B, Hv, K, V), dtype=torch.float32, device=dev)
        problem = _problem(q, k, v, g, b, lengths, scale)
        lib = _abi.load()
        size = lib.rqf_gated_delta_context_bytes(ctypes.byref(problem), int(save))
        if size == ctypes.c_size_t(-1).value:
            raise ValueError(f"gated_delta_scan does not take q {tuple(q.shape)}, v {tuple(v.shape)}")
        context = _scratch(size, dev)
        with torch.cuda.device(dev), _timing.launch("rqf_gated_delta_forward", B * T * Hv,
                                                    _nbytes(q, k, v, g, b, o)):
            _abi.check(lib.rqf_gated_delta_forward(
                ctypes.byref(problem), _abi.ptr(q), _abi.ptr(k), _abi.ptr(v), _abi.ptr(g),
                _abi.ptr(b), _abi.ptr(s0), _abi.ptr(o), _abi.ptr(last), _abi.ptr(context),
                int(save), _abi.stream_of(v)), "rqf_gated_delta_forward")
        _done(dev)
        if save:
            ctx.save_for_backward(q, k, v, g, b, lengths, context)
            ctx.scale = scale
            ctx.has_state = initial_state is not None
        ctx.set_materialize_grads(False)
        return o, last

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_o, grad_last):
        q, k, v, g, b, lengths, context = ctx.saved_tensors
        dev = v.device
        B, T, Hv, V = v.shape
        K = q.shape[-1]
        go = (torch.zeros((B, T, Hv, V), dtype=v.dtype, device=dev) if grad_o is None
              else grad_o.detach().to(v.dtype).contiguous())
        if go.data_ptr() % 16:
            go = go.clone()
        gl = None if grad_last is None else grad_last.detach().float().contiguous()
        dq, dk = (torch.empty(q.shape, dtype=q.dtype, device=dev) for _ in range(2))
        dv = torch.empty((B, T, Hv, V), dtype=v.dtype, device=dev)
        dg, db = (torch.empty((B, T, Hv), dtype=torch.float32, device=dev) for _ in range(2))
        ds0 = (torch.empty((B, Hv, K, V), dtype=torch.float32, device=dev)
               if ctx.has_state and ctx.needs_input_grad[5] else None)
        problem = _problem(q, k, v, g, b, lengths, ctx.scale)
        lib = _abi.load()
        work = _scratch(lib.rqf_gated_delta_backward_workspace_bytes(ctypes.byref(problem)), dev)
        with torch.cuda.device(dev), _timing.launch("rqf_gated_delta_backward", B * T * Hv,
                                                    _nbytes(q, k, v, g, b, go, dq, dk, dv, dg, db)):
            _abi.check(lib.rqf_gated_delta_backward(
                ctypes.byref(problem), _abi.ptr(v), _abi.ptr(context), _abi.ptr(go), _abi.ptr(gl),
                _abi.ptr(dq), _abi.ptr(dk), _abi.ptr(dv), _abi.ptr(dg), _abi.ptr(db),
                _abi.ptr(ds0), _abi.ptr(work), _abi.stream_of(v)), "rqf_gated_delta_backward")
        _done(dev)
        grads = (dq, dk, dv, dg, db, ds0, None, None, None)
        return tuple(x if n else None for x, n in zip(grads, ctx.needs_input_grad))


def gated_delta_scan(q, k, v, log_decay, beta, *, scale: float | None = None, initial_state=None,
                     lengths=None, return_state: bool = False):
    """The gated delta rule over sequences; differentiable in every tensor but lengths.

    q, k           (batch, time, key_heads, K), v (batch, time, value_heads, V), all float32,
                   bfloat16 or float16; value head h reads key head h // (value_heads / key_heads).
                   Views with a dense last axis and rows on 16 bytes are taken as they are.
    log_decay      (batch, time, value_heads), the logarithm of a_t (0 keeps the state, -inf
                   clears it), and beta alike; taken in float32.
    scale          of the output; K ** -0.5 by default.
    initial_state  (batch, value_heads, K, V) float32, or None for zeros.
    lengths        (batch,) integers, or None: what stands past a row's length is not read, its
                   outputs and gradients are 0 and the state there stays as it is.

    Returns o (batch, time, value_heads, V) in v's type, or (o, final_state) with return_state.
    Products are taken to 32-bit accuracy whatever the type (csrc/delta_common.cuh).  While a
    gradient is wanted, the states that enter each 64 tokens are kept for the backward."""
    _check(q, k, v, log_decay, beta, 2)
    B, _, Hv, V = v.shape
    K = q.shape[-1]
    if initial_state is not None:
        _check_state(initial_state, (B, Hv, K, V), "initial_state")
    if lengths is not None:
        if lengths.dtype not in (torch.int32, torch.int64) or tuple(lengths.shape) != (B,):
            raise ValueError(f"lengths must be {B} integers, got {lengths.dtype} {tuple(lengths.shape)}")
        lengths = lengths.to(torch.int64).contiguous()
    scale = K ** -0.5 if scale is None else float(scale)
    args = (q, k, v, log_decay.float(), beta.float(), initial_state)
    _require_cuda(*args, lengths)
    save = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args)
    o, last = _GatedDeltaScan.apply(*args, lengths, scale, save)
    return (o, last) if return_state else o


@torch.no_grad()
def gated_delta_step(q, k, v, log_decay, beta, state, *, slots=None, scale: float | None = None):
    """One token of the gated delta rule for each row of a batch, on states in a pool.

    q, k (batch, key_heads, K), v (batch, value_heads, V), log_decay and beta (batch,
    value_heads) as in gated_delta_scan.  state (pool, value_heads, K, V), dense float32, is
    updated in place: row b works on state[slots[b]], or state[b] without slots.  slots (batch,)
    are distinct integers; a negative one is an idle row, whose output is 0.  One past the pool
    is taken as idle too and raises from check_device_errors().  Returns o (batch, value_heads,
    V) in v's type.  No gradient is recorded."""
    _check(q, k, v, log_decay, beta, 1)
    B, Hv, V = v.shape
    K = q.shape[-1]
    _check_state(state, (state.shape[0] if state.dim() else 0, Hv, K, V), "state")
    if not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError("state must be dense and start on 16 bytes: it is updated in place")
    if slots is None:
        if state.shape[0] < B:
            raise ValueError(f"{B} rows do not fit a pool of {state.shape[0]} states")
    else:
        if slots.dtype not in (torch.int32, torch.int64) or tuple(slots.shape) != (B,):
            raise ValueError(f"slots must be {B} integers, got {slots.dtype} {tuple(slots.shape)}")
        slots = slots.contiguous()
    g, b = log_decay.float(), beta.float()
    dev = _require_cuda(q, k, v, g, b, state, slots)
    q, k, v = (t if t.stride(-1) == 1 else t.contiguous() for t in (q, k, v))
    o = torch.empty((B, Hv, V), dtype=v.dtype, device=dev)
    problem = _problem(q, k, v, g, b, None, K ** -0.5 if scale is None else float(scale))
    lib = _abi.load()
    with torch.cuda.device(dev), _timing.launch("rqf_gated_delta_step", B * Hv,
                                                8 * B * Hv * K * V):
        _abi.check(lib.rqf_gated_delta_step(
            ctypes.byref(problem), _abi.ptr(q), _abi.ptr(k), _abi.ptr(v), _abi.ptr(g),
            _abi.ptr(b), _abi.ptr(slots), int(slots is not None and slots.dtype == torch.int64),
            state.shape[0], _abi.ptr(state), _abi.ptr(o), _abi.stream_of(v)),
            "rqf_gated_delta_step")
    _done(dev)
    return o
