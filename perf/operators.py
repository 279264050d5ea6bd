"""The gated delta rule and gradient clipping as they are measured: cases, inputs, plain forms.

A sequence mixer by the gated delta rule is a recurrence next to this package's
scans, with a K x V matrix for its state.  For each value head, from S_0 on,

    S_t = a_t S_{t-1} + k_t u_t^T,   u_t = beta_t (v_t - (a_t S_{t-1})^T k_t),   a_t = exp(log_decay_t)
    o_t = scale S_t^T q_t

Training and prompts take whole sequences (`gated_delta_scan`), serving takes
one token for each sequence on states that stay in a pool (`gated_delta_step`),
and a training step ends with the norm over all gradients and their clipping
(`global_grad_norm`, `clip_grads_`).

`own` says whose form `run` takes: False the plain one below (torch's
elementary operations in 32 bits), True this package's operators.
"""

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
CHUNK = 64  # tokens that the plain form takes at a time
DEV = "cuda"


# ---------------------------------------------------------------- cases
def listed():
    return [
        # A single short request: latency counts.  161 steps is the feature sequence's length
        # in this repository's first configuration.
        dict(name="scan one short prompt", kind="scan", batch=1, time=161, hk=2, hv=2, k=64, v=64,
             dtype="bfloat16", state=True, lengths=False, train=False),
        # A padded batch of prompts of unlike lengths, empty ones among them, key heads shared.
        dict(name="scan ragged prompts", kind="scan", batch=16, time=2501, hk=2, hv=4, k=64, v=128,
             dtype="float16", state=True, lengths=True, train=False),
        # One long prompt that continues a state: few rows, a long axis.
        dict(name="scan long prompt", kind="scan", batch=1, time=16384, hk=4, hv=8, k=128, v=128,
             dtype="bfloat16", state=True, lengths=False, train=False),
        # Training in 32 bits at odd sizes, through the states at both ends.
        dict(name="train odd fp32", kind="scan", batch=3, time=777, hk=1, hv=3, k=40, v=72,
             dtype="float32", state=True, lengths=True, train=True),
        # Training at the selective configuration's batch and length, width 256 as 4 heads.
        dict(name="train 4096", kind="scan", batch=32, time=4096, hk=4, hv=4, k=64, v=64,
             dtype="bfloat16", state=False, lengths=False, train=True),
        # Training on waveforms of a second, width 256 as 2 heads of 128.
        dict(name="train 16000", kind="scan", batch=32, time=16000, hk=2, hv=2, k=128, v=128,
             dtype="bfloat16", state=False, lengths=False, train=True),
        # Serving: one stream, then many with idle rows, then 32 bits at odd sizes.
        dict(name="step one stream", kind="step", batch=1, pool=4, hk=4, hv=8, k=128, v=128,
             dtype="bfloat16"),
        dict(name="step 256 streams", kind="step", batch=256, pool=320, hk=4, hv=8, k=128, v=128,
             dtype="bfloat16"),
        dict(name="step odd fp32", kind="step", batch=33, pool=40, hk=1, hv=3, k=40, v=72,
             dtype="float32"),
        # The gradients of the encoder that this repository trains (width 256, 6 layers),
        # clipped into a flat buffer as its all-reduce lays one out.
        dict(name="clip encoder", kind="norm", tensors=27, total=1 << 20, dtype="complex64",
             odd=False, clip=True),
        # A model of many small parameters of odd sizes: the buffer's parts start anywhere.
        dict(name="clip many small", kind="norm", tensors=300, total=5_000_003, dtype="float32",
             odd=True, clip=True),
        # A large model's gradients in 16 bits.
        dict(name="clip large", kind="norm", tensors=64, total=400_000_000, dtype="bfloat16",
             odd=False, clip=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    what = rng.choice(["prompt", "prompt", "train", "train", "step", "norm"])
    if what == "norm":
        total = _log(rng, 1 << 14, 300_000_000)
        return dict(kind="norm", tensors=min(_log(rng, 1, 500), total), total=total,
                    dtype=rng.choice(["float32", "bfloat16", "float16", "complex64"]),
                    odd=rng.random() < 0.5, clip=rng.random() < 0.7)
    hk, rep = rng.choice([(1, 1), (2, 1), (4, 1), (1, 3), (2, 2), (4, 2)])
    dims = dict(hk=hk, hv=hk * rep, k=rng.choice([32, 40, 64, 96, 128]),
                v=rng.choice([32, 64, 72, 128]),
                dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]))
    if what == "step":
        batch = _log(rng, 1, 256)
        return dict(kind="step", batch=batch, pool=batch + rng.randint(0, 64), **dims)
    most = 400_000 if what == "train" else 800_000  # tokens of all value heads
    time = _log(rng, 1, 16384)
    batch = _log(rng, 1, max(1, min(64, most // (time * dims["hv"]))))
    return dict(kind="scan", batch=batch, time=time, state=rng.random() < 0.5,
                lengths=rng.random() < 0.4, train=what == "train", **dims)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _unit(x):
    return x / x.norm(dim=-1, keepdim=True)


def _encoder_sizes(total):
    """Six complex layers with their filter leaves and a small head, about `total` elements."""
    n = int(math.isqrt(total // 7))
    return [n * n] * 6 + [n] * 16 + [n * 35, 35, n * n // 2, n, 1]


def _sizes(case):
    if case["dtype"] == "complex64" and case["tensors"] == 27:
        return _encoder_sizes(case["total"])
    n, total = case["tensors"], case["total"]
    # a few large ones, many small ones and odd ones: sizes fall by powers
    w = [1.0 / (1 + i % 17) ** 1.5 for i in range(n)]
    sizes = [max(1, int(total * x / sum(w))) for x in w]
    if case["odd"]:
        sizes[0] += max(0, total - sum(sizes))
        return sizes
    return [-(-n // 64) * 64 for n in sizes]


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "norm":
        dtype = torch.complex64 if case["dtype"] == "complex64" else DTYPES[case["dtype"]]
        sizes = _sizes(case)
        grads = [(torch.randn(n, generator=g, device=DEV, dtype=torch.complex64)
                  if dtype.is_complex else _randn(g, n).to(dtype)) * 1e-2
                 for n in sizes]
        flat = torch.empty(sum(sizes), dtype=dtype, device=DEV) if case["clip"] else None
        return dict(case=case, grads=grads, flat=flat,
                    out=list(flat.split(sizes)) if case["clip"] else None)
    dtype = DTYPES[case["dtype"]]
    b, hk, hv, dk, dv = (case[n] for n in ("batch", "hk", "hv", "k", "v"))
    lead = (b,) if case["kind"] == "step" else (b, case["time"])
    s = dict(case=case)
    s["q"] = _unit(_randn(g, *lead, hk, dk)).to(dtype)
    s["k"] = _unit(_randn(g, *lead, hk, dk)).to(dtype)
    s["v"] = _randn(g, *lead, hv, dv).to(dtype)
    s["log_decay"] = -torch.nn.functional.softplus(_randn(g, *lead, hv) - 4.0)
    s["beta"] = torch.sigmoid(_randn(g, *lead, hv))
    if case["kind"] == "step":
        s["state"] = 0.3 * _randn(g, case["pool"], hv, dk, dv)
        s["slots"] = torch.randperm(case["pool"], generator=g, device=DEV)[:b].to(torch.int32)
        if b > 8:
            s["slots"][3::8] = -1  # idle rows of a serving batch
        return s
    s["initial_state"] = 0.3 * _randn(g, b, hv, dk, dv) if case["state"] else None
    s["lengths"] = None
    if case["lengths"]:
        s["lengths"] = torch.randint(0, case["time"] + 1, (b,), generator=g, device=DEV)
        s["lengths"][0] = case["time"]
        s["lengths"][1:2] = 0
        s["lengths"][2:3] = 1
    if case["train"]:
        s["grad_o"] = _randn(g, *lead, hv, dv).to(dtype)
        s["grad_state"] = 0.3 * _randn(g, b, hv, dk, dv) if case["state"] else None
        for n in ("q", "k", "v", "log_decay", "beta", "initial_state"):
            if s[n] is not None:
                s[n].requires_grad_()
    return s


def work(case):
    if case["kind"] == "norm":
        n = sum(_sizes(case))
        each = {"float32": 4, "bfloat16": 2, "float16": 2, "complex64": 8}[case["dtype"]]
        return {"bytes": n * each * (2 if case["clip"] else 1), "flops": 2 * n + (n if case["clip"] else 0)}
    size = 4 if case["dtype"] == "float32" else 2
    hk, hv, dk, dv = (case[n] for n in ("hk", "hv", "k", "v"))
    token = size * (2 * hk * dk + 2 * hv * dv) + 8 * hv  # q, k, v read, o written; decay and beta
    if case["kind"] == "step":
        return {"bytes": case["batch"] * (token + 8 * hv * dk * dv), "flops": case["batch"] * hv * 7 * dk * dv}
    rows = case["batch"] * case["time"]
    ends = 8 * case["batch"] * hv * dk * dv if case["state"] else 0
    if not case["train"]:
        return {"bytes": rows * token + ends, "flops": rows * hv * 7 * dk * dv}
    # and the output's cotangent read, the five inputs' cotangents written
    grads = size * (2 * hk * dk + 2 * hv * dv) + 8 * hv
    return {"bytes": rows * (token + grads) + 2 * ends, "flops": rows * hv * 21 * dk * dv}


# ---------------------------------------------------------------- plain forms
def _inverse_unit_lower(a):
    """(I + a)^{-1} for strictly lower a (..., 64, 64): inverses of twice the size from two halves."""
    inv = torch.eye(CHUNK, device=a.device, dtype=a.dtype).expand_as(a).clone()
    n = 1
    while n < CHUNK:
        m = CHUNK // (2 * n)
        blocks = lambda x: x.reshape(*x.shape[:-2], m, 2 * n, m, 2 * n).diagonal(dim1=-4, dim2=-2)  # noqa: E731
        low = blocks(a)[..., n:, :n, :].movedim(-1, -3)
        i = blocks(inv)
        i[..., n:, :n, :] = -(i[..., n:, n:, :].movedim(-1, -3) @ low @ i[..., :n, :n, :].movedim(-1, -3)).movedim(-3, -1)
        n *= 2
    return inv


class _Inverse(torch.autograd.Function):
    """The inverse above with its gradient, -T^T g T^T."""

    @staticmethod
    def forward(ctx, a):
        t = _inverse_unit_lower(a)
        ctx.save_for_backward(t)
        return t

    @staticmethod
    def backward(ctx, g):
        (t,) = ctx.saved_tensors
        return -(t.mT @ g @ t.mT)


def _plain_scan(q, k, v, log_decay, beta, scale, state, lengths):
    """Chunks of 64 tokens: inside a chunk u = (I + A)^{-1} beta (v - decayed k S) and
    o = scale (decayed q S + P u) are matrix products over all chunks at once, but for
    what needs the state S that enters the chunk, which one loop over the chunks carries."""
    b, time, hk, dk = q.shape
    hv, dv = v.shape[2:]
    dtype = v.dtype
    q, k, v, log_decay, beta = (x.float() for x in (q, k, v, log_decay, beta))
    if lengths is not None:
        live = (torch.arange(time, device=q.device) < lengths[:, None])[..., None]
        q, k, v = (torch.where(live[..., None], x, 0.0) for x in (q, k, v))
        log_decay, beta = (torch.where(live, x, 0.0) for x in (log_decay, beta))
    n = -(-time // CHUNK)

    def chunks(x):  # (b, time, h, ...) -> (b, h, n, 64, ...)
        x = torch.cat([x, x.new_zeros(b, n * CHUNK - time, *x.shape[2:])], 1)
        return x.reshape(b, n, CHUNK, *x.shape[2:]).movedim(3, 1)

    q, k = (chunks(x).repeat_interleave(hv // hk, 1) for x in (q, k))
    v, log_decay, beta = chunks(v), chunks(log_decay), chunks(beta)
    total = log_decay.cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, device=q.device, dtype=torch.bool).tril()
    decay = torch.where(lower, total[..., :, None] - total[..., None, :], float("-inf")).exp()
    a = (beta[..., None] * decay * (k @ k.mT)).tril(-1)
    t = _Inverse.apply(a) * beta[..., None, :]
    tv, tk = t @ v, t @ (total.exp()[..., None] * k)
    p = scale * decay * (q @ k.mT)
    qd = scale * total.exp()[..., None] * q
    kd = (total[..., -1:] - total).exp()[..., None] * k
    last = total[..., -1].exp()
    s = state if state is not None else q.new_zeros(b, hv, dk, dv)
    out = []
    for i in range(n):
        u = tv[:, :, i] - tk[:, :, i] @ s
        out.append(qd[:, :, i] @ s + p[:, :, i] @ u)
        s = last[:, :, i, None, None] * s + kd[:, :, i].mT @ u
    o = torch.stack(out, 2).movedim(1, 3).reshape(b, n * CHUNK, hv, dv)[:, :time]
    return o.to(dtype), s


def _plain_step(q, k, v, log_decay, beta, scale, state, slots):
    rep = v.shape[1] // q.shape[1]
    q, k = (x.float().repeat_interleave(rep, 1) for x in (q, k))
    live = slots >= 0
    s = state[slots.clamp(min=0)] * log_decay.float().exp()[..., None, None]
    u = beta.float()[..., None] * (v.float() - (s * k[..., None]).sum(-2))
    s = s + k[..., None] * u[..., None, :]
    o = scale * (s * q[..., None]).sum(-2)
    state[slots[live]] = s[live]
    return torch.where(live[:, None, None], o, 0.0).to(v.dtype)


def _plain_norm(grads):
    views = [torch.view_as_real(g) if g.is_complex() else g for g in grads]
    return torch.stack([v.float().square().sum() for v in views]).sum().sqrt()


MAX_NORM = 1.0


def run(s):
    case = s["case"]
    if own:
        import prospective_rqf_b200 as rqf
    if case["kind"] == "norm":
        if s["out"] is None:
            return rqf.global_grad_norm(s["grads"]) if own else _plain_norm(s["grads"])
        if own:
            norm = rqf.clip_grads_(s["grads"], MAX_NORM, out=s["out"])
        else:
            norm = _plain_norm(s["grads"])
            scale = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
            [o.copy_(g * scale if g.is_complex() else g.float() * scale) for o, g in zip(s["out"], s["grads"])]
        return [norm, s["flat"]]
    args = [s[n] for n in ("q", "k", "v", "log_decay", "beta")]
    if case["kind"] == "step":
        if own:
            o = rqf.gated_delta_step(*args, s["state"], slots=s["slots"])
        else:
            o = _plain_step(*args, case["k"] ** -0.5, s["state"], s["slots"])
        return [o, s["state"]]
    with torch.set_grad_enabled(case["train"]):
        if own:
            o, last = rqf.gated_delta_scan(*args, initial_state=s["initial_state"],
                                           lengths=s["lengths"], return_state=True)
        else:
            o, last = _plain_scan(*args, case["k"] ** -0.5, s["initial_state"], s["lengths"])
    if not case["train"]:
        return [o, last]
    if not case["state"]:
        return [o, None, *torch.autograd.grad(o, args, s["grad_o"])]
    grads = torch.autograd.grad([o, last], args + [s["initial_state"]], [s["grad_o"], s["grad_state"]])
    return [o.detach(), last.detach(), *grads]


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_scan(s):
    """Token by token, and back token by token with the states made again for a block at a time."""
    case = s["case"]
    d = lambda n: None if s[n] is None else s[n].detach().double()  # noqa: E731
    q, k, v, g, beta = (d(n).movedim(1, 0) for n in ("q", "k", "v", "log_decay", "beta"))  # time first
    time, b, hk, dk = q.shape
    hv, dv = v.shape[2:]
    rep, scale = hv // hk, dk ** -0.5
    q, k = (x.repeat_interleave(rep, 2) for x in (q, k))
    live = torch.ones(time, b, 1, device=DEV, dtype=torch.float64)
    if s["lengths"] is not None:
        live = (torch.arange(time, device=DEV)[:, None] < s["lengths"]).double()[..., None]
    # a token past its row's length reads and writes nothing and keeps the state
    q, k, v = (x * live[..., None] for x in (q, k, v))
    alpha, beta = torch.exp(g * live), beta * live

    def step(state, t):
        state = state * alpha[t][..., None, None]
        u = beta[t][..., None] * (v[t] - torch.einsum("bhkv,bhk->bhv", state, k[t]))
        return state + k[t][..., None] * u[..., None, :], u

    state = d("initial_state") if case["state"] else torch.zeros(b, hv, dk, dv, device=DEV, dtype=torch.float64)
    block = max(1, min(128, int(2e9 / (state.numel() * 8))))
    entry, o = [], torch.empty_like(v)
    for t in range(time):
        if t % block == 0:
            entry.append(state)
        state, _ = step(state, t)
        o[t] = scale * torch.einsum("bhkv,bhk->bhv", state, q[t])
    last = state
    if not case["train"]:
        return [o.movedim(0, 1), last]
    go = d("grad_o").movedim(1, 0) * live[..., None]
    ds = d("grad_state") if case["state"] else torch.zeros_like(last)
    dq, dk_, dv_ = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dg, db = torch.empty_like(alpha), torch.empty_like(beta)
    for start in reversed(range(0, time, block)):
        before, us, state = [], [], entry[start // block]
        for t in range(start, min(time, start + block)):
            before.append(state)
            state, u = step(state, t)
            us.append(u)
        for t in reversed(range(start, min(time, start + block))):
            prev, u = before.pop(), us.pop()
            decayed = prev * alpha[t][..., None, None]
            after = decayed + k[t][..., None] * u[..., None, :]
            dq[t] = scale * torch.einsum("bhkv,bhv->bhk", after, go[t])
            ds = ds + scale * q[t][..., None] * go[t][..., None, :]
            du = torch.einsum("bhkv,bhk->bhv", ds, k[t])
            dr = beta[t][..., None] * du
            dv_[t] = dr
            db[t] = (du * (v[t] - torch.einsum("bhkv,bhk->bhv", decayed, k[t]))).sum(-1)
            dk_[t] = torch.einsum("bhkv,bhv->bhk", ds, u) - torch.einsum("bhkv,bhv->bhk", decayed, dr)
            ds = ds - k[t][..., None] * dr[..., None, :]
            dg[t] = (ds * decayed).sum((-1, -2))
            ds = ds * alpha[t][..., None, None]
    dq, dk_ = (x.reshape(time, b, hk, rep, dk).sum(3) * live[..., None] for x in (dq, dk_))
    dv_, dg, db = dv_ * live[..., None], dg * live, db * live
    grads = [x.movedim(0, 1) for x in (dq, dk_, dv_, dg, db)]
    return [o.movedim(0, 1), last if case["state"] else None, *grads] + ([ds] if case["state"] else [])


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        total = 0.0
        for g in s["grads"]:
            total += float((torch.view_as_real(g) if g.is_complex() else g).double().pow(2).sum())
        norm = torch.tensor(math.sqrt(total), dtype=torch.float64)
        if s["out"] is None:
            return norm
        c = min(1.0, MAX_NORM / (float(norm) + 1e-6))
        return [norm, torch.cat([(g.to(torch.complex128) if g.is_complex() else g.double()) * c
                                 for g in s["grads"]])]
    if case["kind"] == "scan":
        return _exact_scan(s)
    q, k, v, g, beta = (s[n].double() for n in ("q", "k", "v", "log_decay", "beta"))
    rep, scale = case["hv"] // case["hk"], case["k"] ** -0.5
    state, o = s["state"].double(), torch.zeros_like(v)
    for i, at in enumerate(s["slots"].tolist()):
        if at < 0:
            continue
        for h in range(case["hv"]):
            key, query = k[i, h // rep], q[i, h // rep]
            m = state[at, h] * torch.exp(g[i, h])
            m = m + torch.outer(key, beta[i, h] * (v[i, h] - key @ m))
            state[at, h] = m
            o[i, h] = scale * (query @ m)
    return [o, state]
