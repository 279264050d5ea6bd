"""What the gated delta rule and the gradients' norm refuse, decided before any launch (CPU)."""

import ctypes

import pytest
import torch

import prospective_rqf_b200 as rqf
from prospective_rqf_b200 import _abi


def _args(B=2, T=3, hk=1, hv=2, K=16, V=8, dtype=torch.float32):
    return dict(q=torch.zeros(B, T, hk, K, dtype=dtype), k=torch.zeros(B, T, hk, K, dtype=dtype),
                v=torch.zeros(B, T, hv, V, dtype=dtype), log_decay=torch.zeros(B, T, hv),
                beta=torch.zeros(B, T, hv))


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(2, 3, 16)), "q must have 4 axes"),
    (dict(beta=torch.zeros(2, 3)), "beta must have 3 axes"),
    (dict(k=torch.zeros(2, 3, 2, 16)), "one shape"),
    (dict(v=torch.zeros(2, 4, 2, 8)), "do not match"),
    (dict(v=torch.zeros(2, 3, 2, 8, dtype=torch.bfloat16)), "must all be"),
    (dict(log_decay=torch.zeros(2, 3, 1)), "log_decay must have shape"),
    (dict(beta=torch.zeros(2, 3, 2, dtype=torch.int32)), "floating point"),
    (dict(initial_state=torch.zeros(2, 2, 8, 16)), "initial_state must be float32"),
    (dict(initial_state=torch.zeros(2, 2, 16, 8, dtype=torch.float64)), "initial_state must be float32"),
    (dict(lengths=torch.zeros(2)), "lengths must be 2 integers"),
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), "lengths must be 2 integers"),
    (dict(), "CUDA tensors only"),
])
def test_scan_refuses(change, match):
    args = {**_args(), **change}
    with pytest.raises(RuntimeError if match == "CUDA tensors only" else ValueError, match=match):
        rqf.gated_delta_scan(**args)


@pytest.mark.parametrize("sizes,match", [
    (dict(hk=2, hv=3), "cannot share"), (dict(K=12), "multiples of 8"), (dict(V=4), "multiples of 8"),
    (dict(K=136), "at most 128"), (dict(dtype=torch.float64), "must all be")])
def test_scan_refuses_sizes(sizes, match):
    with pytest.raises(ValueError, match=match):
        rqf.gated_delta_scan(**_args(**sizes))


def _token():
    return {n: t[:, 0] for n, t in _args().items()}


@pytest.mark.parametrize("change,match", [
    (dict(state=torch.zeros(2, 2, 8, 8)), "state must be float32"),
    (dict(state=torch.zeros(1, 2, 16, 8)), "do not fit a pool"),
    (dict(state=torch.zeros(2, 2, 8, 16).transpose(2, 3)), "state must be dense"),
    (dict(slots=torch.zeros(2)), "slots must be 2 integers"),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), "slots must be 2 integers"),
    (dict(q=torch.zeros(2, 1, 1, 16)), "q must have 3 axes"),
    (dict(), "CUDA tensors only"),
])
def test_step_refuses(change, match):
    args = {**_token(), "state": torch.zeros(2, 2, 16, 8), **change}
    with pytest.raises(RuntimeError if match == "CUDA tensors only" else ValueError, match=match):
        rqf.gated_delta_step(**args)


def test_norm_and_clipping_refuse():
    g = torch.zeros(4)
    for call in (lambda x: rqf.global_grad_norm(x), lambda x: rqf.clip_grads_(x, 1.0)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call([g])
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call(g)
        with pytest.raises(ValueError, match="must be float32"):
            call([g.double()])
        with pytest.raises(TypeError, match="must hold tensors"):
            call([1.0])
        with pytest.raises(TypeError):
            call(3)
    with pytest.raises(ValueError, match="negative"):
        rqf.clip_grads_([g], float("nan"))


def test_c_entries_decide_on_the_host():
    """Statuses of the C ABI before any CUDA call: shapes, null pointers, alignment, empty calls."""
    lib = _abi.load()
    p = _abi.DeltaProblem(batch=1, time=70, key_heads=1, value_heads=2, key_dim=64, value_dim=64,
                          dtype=1, scale=1.0)
    size = lib.rqf_gated_delta_context_bytes(ctypes.byref(p), 0)
    assert 0 < size < lib.rqf_gated_delta_context_bytes(ctypes.byref(p), 1) < 1 << 24
    none = [None] * 9
    assert lib.rqf_gated_delta_forward(ctypes.byref(p), *none, 0, None) == 5
    assert lib.rqf_gated_delta_backward(ctypes.byref(p), *[None] * 11) == 5
    assert lib.rqf_gated_delta_step(ctypes.byref(p), *[None] * 6, 0, 4, None, None, None) == 5
    buf = (ctypes.c_char * 64)()
    base = ctypes.addressof(buf)
    ok, odd = base + (-base) % 16, base + (-base) % 16 + 2
    assert lib.rqf_gated_delta_forward(ctypes.byref(p), odd, ok, ok, ok, ok, None, ok, None, ok, 0, None) == 2
    p.q_stride[1] = 4  # 8 bytes
    assert lib.rqf_gated_delta_forward(ctypes.byref(p), ok, ok, ok, ok, ok, None, ok, None, ok, 0, None) == 2
    for name, value, status in (("key_dim", 130, 1), ("key_dim", 12, 1), ("value_dim", -8, 1),
                                ("key_heads", 3, 1), ("time", -1, 1), ("dtype", 3, 5),
                                ("batch", 1 << 40, 1), ("batch", 0, 0)):
        kept = getattr(p, name)
        setattr(p, name, value)
        assert lib.rqf_gated_delta_forward(ctypes.byref(p), *none, 0, None) == status, name
        assert (lib.rqf_gated_delta_context_bytes(ctypes.byref(p), 0) == ctypes.c_size_t(-1).value) == (status != 0)
        setattr(p, name, kept)
    assert lib.rqf_gated_delta_forward(None, *none, 0, None) == 5
    one = (ctypes.c_int64 * 1)(5)
    f32, bad, gone = (ctypes.c_int * 1)(0), (ctypes.c_int * 1)(9), (ctypes.c_void_p * 1)(None)
    assert lib.rqf_global_grad_norm(None, None, None, -1, None, None, None) == 1
    assert lib.rqf_global_grad_norm(gone, one, bad, 1, ok, ok, None) == 5
    assert lib.rqf_global_grad_norm(gone, one, f32, 1, ok, ok, None) == 5
    assert lib.rqf_global_grad_norm((ctypes.c_void_p * 1)(odd), one, f32, 1, ok, ok, None) == 2
    assert lib.rqf_clip_grads((ctypes.c_void_p * 1)(ok), None, one, f32, 1, 1.0, ok, ok, None) == 5
    assert lib.rqf_grad_norm_scratch_bytes(1) >= 8 and lib.rqf_grad_norm_scratch_bytes(2000) > lib.rqf_grad_norm_scratch_bytes(1)
