"""The norm over all gradients of a model, and their clipping, in two launches.

The step between the gradients' all-reduce and the optimiser
(train.py:clip_model_grad_norm_ :777-789), over any number of tensors of mixed
types and sizes.  There is no CPU fallback: other tensors raise.
"""

from __future__ import annotations

import ctypes

import torch

from . import _abi, _timing
from .ops import _done, _require_cuda, _scratch

__all__ = ["global_grad_norm", "clip_grads_"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.complex64: 3}


def _tensors(grads, name: str) -> list[torch.Tensor]:
    if isinstance(grads, torch.Tensor):
        grads = [grads]
    out = [g.detach() for g in grads]
    for g in out:
        if g.dtype not in _DTYPES:
            raise ValueError(f"{name} must be float32, bfloat16, float16 or complex64, got {g.dtype}")
        if g.is_complex() and g.is_conj() or g.is_neg():
            raise ValueError(f"{name} must not be lazy conjugates or negatives: resolve them first")
    return out


def _filled(t: torch.Tensor) -> bool:
    """Whether the tensor's values fill one span of memory, in whatever order of its axes."""
    if t.is_contiguous():
        return True
    span = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != span:
            return False
        span *= size
    return True


def _arrays(ts):
    n = len(ts)
    return ((ctypes.c_void_p * n)(*[t.data_ptr() for t in ts]),
            (ctypes.c_int64 * n)(*[t.numel() for t in ts]),
            (ctypes.c_int * n)(*[_DTYPES[t.dtype] for t in ts]))


@torch.no_grad()
def global_grad_norm(grads) -> torch.Tensor:
    """sqrt(sum |g|^2) over all tensors of `grads` (float32, bfloat16, float16, complex64, mixed as
    they come), as a float32 scalar on their device.  The same tensors give the same bits."""
    ts = _tensors(grads, "grads")
    if not ts:
        return torch.zeros(())
    dev = _require_cuda(*ts)
    ts = [t if _filled(t) else t.contiguous() for t in ts]
    norm = torch.empty((), dtype=torch.float32, device=dev)
    lib = _abi.load()
    scratch = _scratch(lib.rqf_grad_norm_scratch_bytes(len(ts)), dev)
    ptrs, numel, dtypes = _arrays(ts)
    with torch.cuda.device(dev), _timing.launch("rqf_global_grad_norm", sum(numel), 0):
        _abi.check(lib.rqf_global_grad_norm(ptrs, numel, dtypes, len(ts), _abi.ptr(norm),
                                            _abi.ptr(scratch), _abi.stream_of(norm)),
                   "rqf_global_grad_norm")
    _done(dev)
    return norm


@torch.no_grad()
def clip_grads_(grads, max_norm: float, *, out=None) -> torch.Tensor:
    """Scale all tensors of `grads` by min(1, max_norm / (norm + 1e-6)), norm the 2-norm over all
    of them, which is returned as a float32 scalar on their device (no synchronisation).

    In place, or into `out`: tensors of the same shapes, types and orders in memory (parts of an
    optimiser's flat buffer, say), which share no memory with `grads`.  A NaN norm makes all NaN."""
    ts = _tensors(grads, "grads")
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    to = ts if out is None else _tensors(out, "out")
    if len(to) != len(ts):
        raise ValueError(f"{len(ts)} gradients and {len(to)} outputs")
    if not ts:
        return torch.zeros(())
    dev = _require_cuda(*ts, *(() if out is None else to))
    if out is None:
        if len({t.data_ptr() for t in ts if t.numel()}) != sum(1 for t in ts if t.numel()):
            raise ValueError("a tensor stands in grads twice: it would be scaled twice")
    else:
        for t, o in zip(ts, to):
            if o.shape != t.shape or o.dtype != t.dtype:
                raise ValueError(f"out {o.dtype} {tuple(o.shape)} does not match "
                                 f"{t.dtype} {tuple(t.shape)}")
    # what does not lie in memory as its output does goes through a dense copy
    src, dst, back = [], [], []
    for t, o in zip(ts, to):
        if _filled(o) and (o is t or t.stride() == o.stride()):
            src.append(t)
            dst.append(o)
            continue
        c = t.contiguous()
        d = o if o is not t and o.is_contiguous() else c if c.data_ptr() != t.data_ptr() else torch.empty_like(c)
        src.append(c)
        dst.append(d)
        if d is not o:
            back.append((o, d))
    norm = torch.empty((), dtype=torch.float32, device=dev)
    lib = _abi.load()
    scratch = _scratch(lib.rqf_grad_norm_scratch_bytes(len(src)), dev)
    ptrs, numel, dtypes = _arrays(src)
    outs = ptrs if out is None and not back else _arrays(dst)[0]
    with torch.cuda.device(dev), _timing.launch("rqf_clip_grads", sum(numel), 0):
        _abi.check(lib.rqf_clip_grads(ptrs, outs, numel, dtypes, len(src), max_norm,
                                      _abi.ptr(norm), _abi.ptr(scratch), _abi.stream_of(norm)),
                   "rqf_clip_grads")
    _done(dev)
    for o, d in back:
        o.copy_(d)
    return norm
