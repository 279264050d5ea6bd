"""The norm over all gradients and their clipping, on the GPU."""

import math

import pytest
import torch

import prospective_rqf_b200 as rqf

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.complex64]
# The norm is a sum of squares, eight at a time in 32 bits (8 x 2^-24 each at most, and the
# root halves it) and in 64 from there on, rounded once; the factor is two roundings more,
# and the product one in the tensor's own type.
NORM_TOL = 8 * 2.0 ** -24
FACTOR_TOL = NORM_TOL + 3 * 2.0 ** -24
ROUNDOFF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11,
            torch.complex64: 2.0 ** -24}


def _rand(n, dtype, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, generator=g, dtype=dtype if dtype.is_complex else torch.float32) * size
    return x.to(dtype).cuda()


def _wide(t):
    return torch.view_as_real(t.to(torch.complex128)) if t.is_complex() else t.double()


def _norm(ts):
    return math.sqrt(sum(float((_wide(t.detach()) ** 2).sum()) for t in ts))


def _check(grads, max_norm, out=None):
    want = _norm(grads)
    c = min(1.0, max_norm / (want + 1e-6))
    expected = [_wide(g) * c for g in grads]
    assert abs(float(rqf.global_grad_norm(grads)) - want) <= NORM_TOL * want
    norm = rqf.clip_grads_(grads, max_norm, out=out)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - want) <= NORM_TOL * want
    for g, e in zip(grads if out is None else out, expected):
        tiny = 2.0 ** -25 if g.dtype == torch.float16 else 0.0  # half's subnormals
        bound = (ROUNDOFF[g.dtype] + FACTOR_TOL) * e.abs() * 1.01 + tiny
        assert bool(((_wide(g) - e).abs() <= bound).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[1], [7], [1, 2, 3, 0, 5], [4096, 4097, 8191], [100_003, 16, 1]])
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_types_and_sizes(dtype, sizes, max_norm):
    _check([_rand(n, dtype, i) for i, n in enumerate(sizes)], max_norm)
    grads = [_rand(n, dtype, i) for i, n in enumerate(sizes)]
    _check(grads, max_norm, out=[torch.full_like(g, math.nan) for g in grads])


def test_types_side_by_side():
    _check([_rand(1000 + i, TYPES[i % 4], i) for i in range(12)], 1.0)


@pytest.mark.parametrize("n", [31, 33, 119, 121, 959, 961, 2500])
def test_many_tensors(n):
    """On both sides of the sizes at which the table of tensors changes."""
    grads = [_rand(1 + 37 * i % 300, TYPES[i % 4], i) for i in range(n)]
    flat = [torch.empty_like(g) for g in grads]
    _check(grads, 1.0, out=flat)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset_in,offset_out", [(0, 1), (1, 0), (3, 3), (1, 2), (5, 7)])
def test_parts_of_buffers_at_any_offset(dtype, offset_in, offset_out):
    n = 20_011
    src = _rand(n + 16, dtype, 1)
    dst = torch.full_like(src, 3.0)
    grads, out = [src[offset_in:offset_in + n]], [dst[offset_out:offset_out + n]]
    _check(grads, 2.0, out=out)
    rest = torch.ones(n + 16, dtype=torch.bool)
    rest[offset_out:offset_out + n] = False
    assert bool((dst[rest.cuda()] == 3.0).all())  # nothing else was written


def test_orders_in_memory():
    a = _rand(60 * 70, torch.float32, 1).view(60, 70)
    turned, holes = a.t().clone().t(), _rand(60 * 140, torch.float32, 2).view(60, 140)[:, ::2]
    spread = _rand(64, torch.float32, 3)[:1].expand(50)  # one value fifty times
    kept = holes.clone()
    want = _norm([turned, holes, spread])
    assert abs(float(rqf.global_grad_norm([turned, holes, spread])) - want) <= NORM_TOL * want
    _check([turned, holes], 1.0)
    assert not torch.equal(holes, kept)
    grads = [a.clone().t(), kept.clone()]
    _check(grads, 1.0, out=[torch.zeros(70, 60, device="cuda"), torch.zeros(140, 60, device="cuda").t()[:, ::2]])


def test_sizes_of_values():
    """Squares that leave 32 bits' range at either end."""
    _check([_rand(5000, torch.float32, 1, 1e25), _rand(100, torch.float32, 2)], 1.0)
    big = rqf.global_grad_norm([_rand(5000, torch.float32, 1, 1e25)])
    assert math.isfinite(float(big))
    tiny = [_rand(5000, torch.float32, 1, 1e-30)]
    want = _norm(tiny)
    assert abs(float(rqf.global_grad_norm(tiny)) - want) <= NORM_TOL * want
    zeros = [torch.zeros(100, device="cuda")]
    assert float(rqf.clip_grads_(zeros, 1.0)) == 0.0 and not zeros[0].any()


def test_values_that_are_not_finite():
    g = [_rand(100, torch.float32, 1), _rand(100, torch.bfloat16, 2)]
    g[0][3] = math.inf
    out = [torch.empty_like(x) for x in g]
    assert float(rqf.clip_grads_(g, 1.0, out=out)) == math.inf
    assert math.isnan(float(out[0][3])) and int(torch.isnan(out[0]).sum()) == 1 and not out[1].any()
    g[1][5] = math.nan
    assert math.isnan(float(rqf.clip_grads_(g, 1.0, out=out)))
    assert all(bool(torch.isnan(x).all()) for x in out)


def test_same_bits_each_time_and_on_another_stream():
    grads = [_rand(50_021, TYPES[i % 4], i) for i in range(40)]
    first = rqf.global_grad_norm(grads)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = rqf.global_grad_norm(grads)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    version = grads[0]._version
    rqf.clip_grads_(grads, 1.0)
    assert grads[0]._version > version


def test_in_a_graph():
    grads = [_rand(10_000, torch.float32, i) for i in range(3)]
    out = [torch.empty_like(g) for g in grads]
    want = rqf.clip_grads_(grads, 1.0, out=out)
    kept = [o.clone() for o in out]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = rqf.clip_grads_(grads, 1.0, out=out)
    for o in out:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(out, kept))


def test_refusals_on_the_gpu():
    g = _rand(8, torch.float32, 1)
    with pytest.raises(ValueError, match="twice"):
        rqf.clip_grads_([g, g], 1.0)
    with pytest.raises(ValueError, match="does not match"):
        rqf.clip_grads_([g], 1.0, out=[g[:4]])
    with pytest.raises(ValueError, match="outputs"):
        rqf.clip_grads_([g], 1.0, out=[])
    with pytest.raises(ValueError, match="negative"):
        rqf.clip_grads_([g], -1.0)
    with pytest.raises(ValueError, match="conjugates"):
        rqf.global_grad_norm([_rand(4, torch.complex64, 1).conj()])
    assert float(rqf.global_grad_norm([])) == 0.0
