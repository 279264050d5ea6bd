"""The gated delta rule on the GPU against its definition in 64 bits."""

import math

import pytest
import torch

import prospective_rqf_b200 as rqf
from _delta_ref import TOL32, assert_near, inputs, reference

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = ("q", "k", "v", "log_decay", "beta", "initial_state")


def _state(B, hv, K, V, seed=9):
    return 0.5 * torch.randn(B, hv, K, V, generator=torch.Generator().manual_seed(seed)).cuda()


def _check(args, state=None, lengths=None, scale=None, tol=TOL32, skip=()):
    """Forward and all gradients against the reference's."""
    leaves = [t.detach().clone().requires_grad_() for t in args]
    s0 = None if state is None else state.clone().requires_grad_()
    o, last = rqf.gated_delta_scan(*leaves, scale=scale, initial_state=s0, lengths=lengths,
                                   return_state=True)
    exact = [t.detach().double().requires_grad_() for t in args]
    e0 = None if state is None else state.double().requires_grad_()
    eo, elast = reference(*exact, scale=scale, initial_state=e0, lengths=lengths)
    assert_near(o.detach(), eo.detach(), "o", tol)
    assert_near(last.detach(), elast.detach(), "final state", tol)
    g = torch.Generator().manual_seed(77)
    go = torch.randn(o.shape, generator=g).to(o.dtype).cuda()
    gs = torch.randn(last.shape, generator=g).cuda()
    wrt, ewrt = leaves + [s0] * (s0 is not None), exact + [e0] * (e0 is not None)
    got = torch.autograd.grad([o, last], wrt, [go, gs])
    want = torch.autograd.grad([eo, elast], ewrt, [go.double(), gs.double()])
    for n, a, b in zip(NAMES, got, want):
        if n not in skip:
            assert_near(a, b, f"gradient of {n}", tol)
    rqf.check_device_errors()


@pytest.mark.parametrize("T", [1, 2, 15, 63, 64, 65, 129, 200])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_lengths_of_the_sequence(T, dtype):
    _check(inputs(2, T, 1, 2, 64, 64, dtype, seed=T), _state(2, 2, 64, 64))


@pytest.mark.parametrize("hk,hv,K,V", [(1, 1, 8, 8), (2, 2, 16, 24), (1, 3, 24, 40), (2, 2, 32, 128),
                                       (1, 1, 40, 72), (2, 4, 64, 16), (1, 1, 72, 64), (1, 2, 96, 96),
                                       (1, 1, 128, 128), (1, 1, 120, 136), (3, 3, 128, 200)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_head_sizes(hk, hv, K, V, dtype):
    _check(inputs(2, 130, hk, hv, K, V, dtype, seed=K + V))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("K,V", [(32, 128), (64, 128), (128, 128)])
def test_many_heads_take_the_wider_ctas(dtype, K, V):
    """Enough heads that the pass over the chunks has eight warps to a CTA."""
    _check(inputs(10, 70, 4, 8, K, V, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_unlike_lengths(dtype):
    """Rows that end early read nothing past their end (NaN there), give zeros, keep the state."""
    lengths = torch.tensor([0, 1, 64, 65, 150, 7])
    args = inputs(6, 150, 2, 4, 64, 64, dtype)
    _check(args, _state(6, 4, 64, 64), lengths.cuda())
    clean = [t.clone() for t in args]
    for t in args:
        for b, n in enumerate(lengths.tolist()):
            t[b, n:] = math.nan
    state = _state(6, 4, 64, 64)
    want = rqf.gated_delta_scan(*clean, initial_state=state, lengths=lengths.cuda(), return_state=True)
    leaves = [t.requires_grad_() for t in args]
    o, last = rqf.gated_delta_scan(*leaves, initial_state=state, lengths=lengths.to(torch.int32).cuda(),
                                   return_state=True)
    assert torch.equal(o, want[0]) and torch.equal(last, want[1])
    assert torch.equal(last[0], state[0])
    grads = torch.autograd.grad(o, leaves, torch.ones_like(o))
    for n, t in zip(NAMES, grads):
        assert bool(torch.isfinite(t).all()), n
        for b, m in enumerate(lengths.tolist()):
            assert not t[b, m:].any(), n
    for b, m in enumerate(lengths.tolist()):
        assert not o[b, m:].any()


@pytest.mark.parametrize("dtype,hv,K,V,T", [(F32, 1, 40, 24, 1000), (BF16, 2, 128, 128, 833), (F16, 2, 64, 72, 769)])
@pytest.mark.parametrize("lengths", [None, [0, 1], [700, 64], [257, 769]])
def test_few_rows_over_long_sequences(dtype, hv, K, V, T, lengths):
    """Long sequences of few rows are cut into spans, of which short rows leave some empty."""
    n = None if lengths is None else torch.tensor(lengths).cuda()
    _check(inputs(2, T, 1, hv, K, V, dtype, decay=5.0), _state(2, hv, K, V), n)


def test_lengths_out_of_range_are_taken_into_range():
    args = inputs(2, 70, 1, 1, 32, 32, F32)
    full = rqf.gated_delta_scan(*args, lengths=torch.tensor([70, 0]).cuda())
    assert torch.equal(rqf.gated_delta_scan(*args, lengths=torch.tensor([1 << 40, -5]).cuda()), full)


def test_empty_calls():
    for B, T in ((0, 5), (2, 0), (0, 0)):
        args = inputs(B, T, 1, 2, 16, 16, F32)
        state = _state(B, 2, 16, 16)
        o, last = rqf.gated_delta_scan(*args, initial_state=state, return_state=True)
        assert o.shape == (B, T, 2, 16) and torch.equal(last, state)
    leaves = [t.requires_grad_() for t in inputs(2, 0, 1, 2, 16, 16, F32)]
    state = _state(2, 2, 16, 16).requires_grad_()
    _, last = rqf.gated_delta_scan(*leaves, initial_state=state, return_state=True)
    (g,) = torch.autograd.grad(last, [state], torch.full_like(last, 2.0))
    assert torch.equal(g, torch.full_like(last, 2.0))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_of_one_projection(dtype):
    """q, k and v as parts of one tensor, batch and time exchanged, and an odd offset: strides
    that the kernels take as they are, and ones that are copied first."""
    B, T, h, K = 2, 100, 2, 64
    q, k, v, g, b = inputs(B, T, h, h, K, K, dtype)
    want = rqf.gated_delta_scan(q, k, v, g, b)
    packed = torch.cat([q, k, v], -1)
    views = packed.split(K, -1)
    assert torch.equal(rqf.gated_delta_scan(*views, g, b), want)
    swapped = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, g, b)]
    assert torch.equal(rqf.gated_delta_scan(*swapped), want)
    heads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, g, b)]
    assert torch.equal(rqf.gated_delta_scan(*heads), want)
    shifted = []
    for t in (q, k, v):
        flat = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape)
        flat.copy_(t)
        shifted.append(flat)
    assert torch.equal(rqf.gated_delta_scan(*shifted, g, b), want)
    last_axis = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]
    assert torch.equal(rqf.gated_delta_scan(*last_axis, g, b), want)
    shared = [t[:, :, :1].expand(B, T, h, K) for t in (q, k)]  # broadcast heads
    a = rqf.gated_delta_scan(*shared, v, g, b)
    assert torch.equal(a, rqf.gated_delta_scan(q[:, :, :1], k[:, :, :1], v, g, b))


def test_gradients_of_broadcast_inputs():
    """A gate for all heads and a key for the whole batch: gradients summed over what shares them."""
    q, k, v, g, b = inputs(3, 66, 2, 2, 32, 32, F32)
    g1, k1 = g[..., :1].clone().requires_grad_(), k[:1].clone().requires_grad_()
    o = rqf.gated_delta_scan(q, k1.expand_as(k), v, g1.expand_as(g), b)
    go = torch.randn_like(o)
    got = torch.autograd.grad(o, [g1, k1], go)
    eg, ek = g1.detach().double().requires_grad_(), k1.detach().double().requires_grad_()
    eo, _ = reference(q, ek.expand(k.shape), v, eg.expand(g.shape), b)
    for n, a, w in zip(("log_decay", "k"), got, torch.autograd.grad(eo, [eg, ek], go.double())):
        assert_near(a, w, n)


def test_cotangents_that_are_absent_or_strided():
    args = inputs(2, 80, 1, 2, 32, 32, F32)
    state = _state(2, 2, 32, 32)

    def both(pick):
        leaves = [t.clone().requires_grad_() for t in (*args, state)]
        exact = [t.double().requires_grad_() for t in (*args, state)]
        got = pick(*rqf.gated_delta_scan(*leaves[:5], initial_state=leaves[5], return_state=True))
        want = pick(*reference(*exact[:5], initial_state=exact[5]))
        for n, a, w in zip(NAMES, torch.autograd.grad(got, leaves, allow_unused=True),
                           torch.autograd.grad(want, exact, allow_unused=True)):
            assert_near(a, torch.zeros_like(a, dtype=torch.float64) if w is None else w, n)

    both(lambda o, s: o.sum())            # a cotangent with strides of 0
    both(lambda o, s: s.sum())            # none for o
    both(lambda o, s: (o[:, ::2] ** 2).sum())


def test_only_the_gradients_that_are_wanted():
    args = inputs(1, 40, 1, 1, 16, 16, F32)
    v = args[2].requires_grad_()
    o = rqf.gated_delta_scan(*args)
    (g,) = torch.autograd.grad(o.sum(), [v])
    assert g.shape == v.shape and rqf.gated_delta_scan(*[t.detach() for t in args]).requires_grad is False
    with torch.no_grad():
        assert not rqf.gated_delta_scan(*args).requires_grad
    # gates in 16 bits get gradients of their type
    b = args[4].to(BF16).requires_grad_()
    o = rqf.gated_delta_scan(*args[:4], b)
    assert torch.autograd.grad(o.sum(), [b])[0].dtype == BF16


def test_gradient_against_differences():
    """Derivatives along a direction of all inputs together, by central differences of the
    definition in 64 bits (error about 1e-10 of its value)."""
    args = inputs(1, 90, 1, 2, 24, 16, F32)
    state = _state(1, 2, 24, 16)
    g = torch.Generator().manual_seed(5)
    along = [torch.randn(t.shape, generator=g, dtype=torch.float64).cuda() for t in (*args, state)]
    w = torch.randn(1, 90, 2, 16, generator=g).cuda()
    ws = torch.randn(1, 2, 24, 16, generator=g).cuda()

    def value(eps):
        x = [t.double() + eps * d for t, d in zip((*args, state), along)]
        o, s = reference(*x[:5], initial_state=x[5])
        return float((o * w).sum() + (s * ws).sum())

    want = (value(1e-5) - value(-1e-5)) / 2e-5
    leaves = [t.clone().requires_grad_() for t in (*args, state)]
    o, s = rqf.gated_delta_scan(*leaves[:5], initial_state=leaves[5], return_state=True)
    grads = torch.autograd.grad([o, s], leaves, [w, ws])
    got = sum(float((a.double() * d).sum()) for a, d in zip(grads, along))
    size = math.sqrt(sum(float(a.double().norm() ** 2) for a in grads)) * math.sqrt(
        sum(float(d.norm() ** 2) for d in along))
    assert abs(got - want) <= TOL32 * size


# ---------------------------------------------------------------- values at their edges
def test_gates_that_clear_or_keep():
    """log_decay of -inf (a cleared state), very negative ones and exact 0."""
    args = inputs(2, 140, 1, 2, 32, 32, F32)
    args[3][:, 5] = -math.inf
    args[3][:, 70:72] = -math.inf
    args[3][:, 100] = -1e30
    args[3][:, 20:40] = 0.0
    state = _state(2, 2, 32, 32)
    leaves = [t.clone().requires_grad_() for t in args]
    o, last = rqf.gated_delta_scan(*leaves, initial_state=state, return_state=True)
    eo, elast = reference(*args, initial_state=state)
    assert_near(o.detach(), eo, "o")
    assert_near(last.detach(), elast, "state")
    grads = torch.autograd.grad(o.sum(), leaves)
    assert all(bool(torch.isfinite(t).all()) for t in grads)
    assert not grads[3][:, 5].any() and not grads[3][:, 100].any()


def test_a_closed_gate_parts_large_values_from_small_ones():
    """Two documents in one row, the first with values ten thousand times the second's: the second's
    gradients are as exact as if it stood alone."""
    args = inputs(1, 150, 1, 2, 32, 32, F32)
    args[2][:, :40] *= 1e4
    args[3][:, 40] = -math.inf
    go = torch.randn(1, 150, 2, 32, generator=torch.Generator().manual_seed(3)).cuda()
    leaves = [t.clone().requires_grad_() for t in args]
    grads = torch.autograd.grad(rqf.gated_delta_scan(*leaves), leaves, go)
    alone = [t[:, 40:].double().requires_grad_() for t in args]
    want = torch.autograd.grad(reference(*alone)[0], alone, go[:, 40:].double())
    for n, a, b in zip(NAMES, grads, want):
        assert_near(a[:, 40:], b, f"gradient of {n}")


def test_keys_that_are_alike():
    """Equal keys with beta = 1 and no decay: the inverse inside a chunk has entries that cancel."""
    args = inputs(1, 128, 1, 1, 32, 32, F32)
    args[1][:] = args[1][:, :1]
    args[3][:] = 0.0
    args[4][:] = 1.0
    _check(args, skip=("log_decay",))
    # Here the state is one key's value, the next token's cotangent passes none of it, and the
    # gradient of log_decay is 0: what is left is the rounding of terms of the others' size.
    leaves = [t.clone().requires_grad_() for t in args]
    o = rqf.gated_delta_scan(*leaves)
    grads = torch.autograd.grad(o, leaves, torch.randn(o.shape, generator=torch.Generator().manual_seed(77)).cuda())
    assert float(grads[3].norm()) <= TOL32 * max(float(g.norm()) for g in grads)
    args[1][:, ::2] = -args[1][:, ::2]
    args[4][:] = 1.9
    o, _ = reference(*args)
    assert_near(rqf.gated_delta_scan(*args), o, "o")


@pytest.mark.parametrize("size", [1e-18, 1e-6, 300.0, 1e10])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_keys_and_values_of_any_size(size, dtype):
    """Rows are scaled before they become halves: large and small ones keep their bits, side by side."""
    q, k, v, g, b = inputs(2, 100, 1, 1, 64, 64, dtype)
    q[:, ::3] *= size
    v[:, 1::2] *= size
    k[:, ::2] *= min(size, 1.0)
    _check([q, k, v, g, b])


def test_zero_keys_and_beta():
    q, k, v, g, b = inputs(1, 100, 1, 2, 32, 32, F32)
    k[:, 3:9] = 0.0
    q[:, 50] = 0.0
    b[:, 60:70] = 0.0
    v[:, 80] = 0.0
    _check([q, k, v, g, b], _state(1, 2, 32, 32))
    zero = [torch.zeros_like(t) for t in (q, k, v, g, b)]
    assert not rqf.gated_delta_scan(*zero).any()


def test_a_value_that_is_not_finite_stays_in_its_column():
    q, k, v, g, b = inputs(1, 130, 1, 1, 32, 32, F32)
    v[0, 70, 0, 3] = math.nan
    o = rqf.gated_delta_scan(q, k, v, g, b)
    bad = torch.isnan(o[0, :, 0])
    assert bad[70:, 3].all() and not bad[:64].any()
    bad[:, 3] = False
    assert not bad.any()


# ---------------------------------------------------------------- calls in a program
def test_parts_of_a_sequence_through_the_state():
    args = inputs(2, 200, 1, 2, 64, 64, F32)
    whole, last = rqf.gated_delta_scan(*args, return_state=True)
    state, parts = None, []
    for a, b in ((0, 1), (1, 65), (65, 70), (70, 200)):
        o, state = rqf.gated_delta_scan(*[t[:, a:b] for t in args], initial_state=state, return_state=True)
        parts.append(o)
    assert_near(torch.cat(parts, 1), whole.double(), "o", 2 * TOL32)
    assert_near(state, last.double(), "state", 2 * TOL32)


def test_same_call_same_bits_on_another_stream_and_in_a_graph():
    args = [t.requires_grad_() for t in inputs(3, 150, 2, 4, 64, 128, BF16)]

    def once():
        o = rqf.gated_delta_scan(*args)
        return (o, *torch.autograd.grad(o, args, torch.ones_like(o)))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    still = [t.detach() for t in args]
    with torch.cuda.graph(graph):
        o = rqf.gated_delta_scan(*still)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, first[0])


# ---------------------------------------------------------------- one token
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hk,hv,K,V", [(1, 1, 8, 8), (1, 3, 40, 72), (2, 4, 64, 64), (2, 2, 128, 128),
                                       (1, 1, 120, 200)])
def test_step_against_the_definition(dtype, hk, hv, K, V):
    B = 5
    args = inputs(B, 3, hk, hv, K, V, dtype)
    pool = _state(9, hv, K, V)
    slots = torch.tensor([4, 0, -1, 8, 2], dtype=torch.int32).cuda()
    want, untouched = pool.clone(), [1, 3, 5, 6, 7]
    before = pool.clone()
    for t in range(3):
        o = rqf.gated_delta_step(*[x[:, t] for x in args], pool, slots=slots)
        live = slots >= 0
        eo, es = reference(*[x[live][:, t:t + 1] for x in args], initial_state=want[slots[live].long()])
        assert_near(o[live], eo[:, 0], "o")
        assert not o[~live].any()
        want[slots[live].long()] = es.float()
    assert_near(pool[slots[live].long()], es, "state")
    assert torch.equal(pool[untouched], before[untouched])
    rqf.check_device_errors()


def test_step_continues_a_scan():
    args = inputs(4, 70, 2, 4, 64, 64, BF16)
    _, state = rqf.gated_delta_scan(*[t[:, :69] for t in args], return_state=True)
    whole, last = rqf.gated_delta_scan(*args, return_state=True)
    o = rqf.gated_delta_step(*[t[:, 69] for t in args], state)
    assert_near(o, whole[:, 69].double(), "o", 2 * TOL32 + 2.0 ** -8)
    assert_near(state, last.double(), "state", 2 * TOL32)


def test_step_takes_any_strides_and_both_index_types():
    B, h, K = 3, 2, 32
    args = inputs(B, 2, h, h, K, K, BF16)
    tokens = [t[:, 1] for t in args]
    a, b, c = (_state(4, h, K, K) for _ in range(3))
    slots = torch.tensor([3, 1, 0])
    want = rqf.gated_delta_step(*[t.contiguous() for t in tokens], a, slots=slots.cuda())
    assert torch.equal(rqf.gated_delta_step(*tokens, b, slots=slots.to(torch.int32).cuda()), want)
    wide = [torch.empty(B, h, 2 * K + 1, dtype=BF16, device="cuda")[..., 1:K + 1].copy_(t) for t in tokens[:3]]
    assert torch.equal(rqf.gated_delta_step(*wide, *tokens[3:], c, slots=slots.cuda()), want)
    assert torch.equal(a, b) and torch.equal(a, c)


def test_step_refuses_a_slot_past_the_pool():
    """It is an idle row, and the device's error word says so."""
    args = [t[:, 0] for t in inputs(2, 1, 1, 1, 16, 16, F32)]
    pool = _state(2, 1, 16, 16)
    before = pool.clone()
    o = rqf.gated_delta_step(*args, pool, slots=torch.tensor([2, 1], dtype=torch.int32).cuda())
    assert not o[0].any() and torch.equal(pool[0], before[0]) and not torch.equal(pool[1], before[1])
    with pytest.raises(rqf.RQFError):
        rqf.check_device_errors()
    rqf.check_device_errors()


def test_step_in_a_graph_and_version_counter():
    args = [t[:, 0].contiguous() for t in inputs(2, 1, 1, 1, 64, 64, BF16)]
    pool = _state(2, 1, 64, 64)
    start = pool.clone()
    version = pool._version
    want = rqf.gated_delta_step(*args, pool)
    assert pool._version > version
    after = pool.clone()
    pool.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = rqf.gated_delta_step(*args, pool)
    pool.copy_(start)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, want) and torch.equal(pool, after)
