"""The norm over all gradients of a model, and their clipping, in two launches.

The step between the gradients' all-reduce and the optimiser
(train.py:clip_model_grad_norm_ :777-789), over any number of tensors of mixed
types and sizes.  There is no CPU fallback: other tensors raise.
"""

from __future__ import annotations

import torch

from . import _abi
from .ops import _done

__all__ = ["global_grad_norm", "clip_grads_"]


def global_grad_norm(grads) -> torch.Tensor:
    """sqrt(sum |g|^2) over all tensors of `grads` (float32, bfloat16, float16, complex64, mixed as
    they come), as a float32 scalar on their device.  The same tensors give the same bits."""
    norm = _abi.native().grad_norm(grads)
    _done(norm.device)
    return norm


def clip_grads_(grads, max_norm: float, *, out=None) -> torch.Tensor:
    """Scale all tensors of `grads` by min(1, max_norm / (norm + 1e-6)), norm the 2-norm over all
    of them, which is returned as a float32 scalar on their device (no synchronisation).

    In place, or into `out`: tensors of the same shapes and types (parts of an optimiser's flat
    buffer, say), which share no memory with `grads`.  A NaN norm makes all NaN."""
    norm = _abi.native().clip_grads(grads, max_norm, out)
    _done(norm.device)
    return norm
