"""The gated delta rule token by token in 64 bits, from its definition."""

import torch


def reference(q, k, v, log_decay, beta, scale=None, initial_state=None, lengths=None):
    """o and the final state, differentiable; any device, computed in float64."""
    B, T, hk, K = q.shape
    hv, V = v.shape[2:]
    rep = hv // hk
    scale = K ** -0.5 if scale is None else scale
    q, k = (x.double().repeat_interleave(rep, 2) for x in (q, k))
    v, log_decay, beta = v.double(), log_decay.double(), beta.double()
    S = (torch.zeros(B, hv, K, V, dtype=torch.float64, device=q.device) if initial_state is None
         else initial_state.double())
    out = []
    for t in range(T):
        a = torch.exp(log_decay[:, t])[..., None, None]
        D = a * S
        u = beta[:, t][..., None] * (v[:, t] - torch.einsum("bhkv,bhk->bhv", D, k[:, t]))
        N = D + torch.einsum("bhk,bhv->bhkv", k[:, t], u)
        o = scale * torch.einsum("bhkv,bhk->bhv", N, q[:, t])
        if lengths is not None:
            on = (t < lengths).view(B, 1, 1)
            N = torch.where(on[..., None], N, S)
            o = torch.where(on, o, torch.zeros_like(o))
        S = N
        out.append(o)
    o = torch.stack(out, 1) if out else v.new_zeros(B, 0, hv, V)
    return o, S


def inputs(B, T, hk, hv, K, V, dtype, seed=0, decay=3.0, device="cuda"):
    """Unit keys and queries, decays from strong to weak, as a model has them."""
    g = torch.Generator().manual_seed(seed)
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    q, k = (unit(torch.randn(B, T, hk, K, generator=g)).to(dtype) for _ in range(2))
    v = torch.randn(B, T, hv, V, generator=g).to(dtype)
    log_decay = -torch.nn.functional.softplus(torch.randn(B, T, hv, generator=g) - decay)
    beta = torch.sigmoid(torch.randn(B, T, hv, generator=g))
    return [x.to(device) for x in (q, k, v, log_decay, beta)]


# What a result may be off.  32-bit ones: products are sums of up to 128 terms whose
# additions each lose at most 2^-23 of the running sum, which bounds the error of one
# product by 128 x 2^-23 of its magnitude, and the decays keep the chunks' errors from
# adding up.  16-bit ones: their unit roundoff besides.
TOL32 = 128 * 2.0 ** -23
ROUNDOFF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def assert_near(got, want, what, tol=TOL32):
    """The 2-norm of the error beyond the type's own rounding, over the result's."""
    assert got.shape == want.shape, what
    want = want.to(got.device)
    err = (got.double() - want).abs() - ROUNDOFF[got.dtype] * want.abs()
    norm = float(want.norm())
    rel = float(err.clamp(min=0).norm()) / norm if norm else float(got.double().norm())
    assert rel <= tol, f"{what}: {rel:.2e} > {tol:.2e}"
