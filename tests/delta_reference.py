"""The gated delta rule in 64 bits, token by token, with error bars (tests of the gated delta operators).

Bars.  With |k| <= 1 and beta <= 1 a token multiplies the state's columns by a (I - beta k k^T), of norm at most a, so an
error E in a column's 2-norm goes to a E, and what the token's own arithmetic adds is a few units of rounding of the
column and of what is written: E_t = a_t E_{t-1} + kappa u (|C_t| + |beta d| |k|).  A token of the recurrent kernel sums DQK
values in float32, DQK / 32 of them one after another, then in trees: kappa u = (DQK / 32 + 16) 2^-24.  The chunkwise
kernels round operands to pairs of f16 (2^-22): the state, R, T, U and U's decayed copy, once each (5), the products
drop lo lo (3 of them, below 2^-22 each), and up to 320 float32 sums of 2^-24 come to sqrt(320) 2^-24 = 4.5 2^-22: kappa u = 16
2^-22, rounded up.  h is off by scale |q| E and, where its operands are single f16 planes (bf16 in and out), by half a unit (2^-11) of the
state's, P's and U's values: 2^-11 scale (|q| max |C| + 2 sum_j D_ij |q_i.k_j| |U_j|); and by its own rounding.

Within a chunk the operands are the state at its start (decayed, c_t C_0) and v - c_t k C_0: the corrections that shrink
C_0 to C_t are sums of terms of that size, rounded at that size.  So |C_t| above is max(|C_t|, c_t |C_0|) there (``chunk``).
f16 ends at 2^-24: an operand whose largest value stands at 2^14 or more is off by 2^-39 of that in its small ones too.
There are 4 (state, R, U, its decayed copy), and up to 64 tokens' of them are summed with factors up to 1: 64 x 4 x 2^-39 =
2^-31 of the largest column of the chunk's start, were they all of one sign; sqrt(64) of them, 2^-34, is taken.
"""

import torch

CHUNK_KU = 16 * 2.0 ** -22


def recurrent_ku(DQK):
    return (DQK / 32 + 16) * 2.0 ** -24


def make(B, NH, NHK, S, DQK, DV, dtype, gate, seed, state=True, device="cuda:0", strong=False):
    """Inputs as the models make them: q and k of length at most 1, decays of many time constants."""
    r = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=r)  # noqa: E731
    q, k = n(B, NHK, S, DQK), n(B, NHK, S, DQK) + 0.7 * n(B, NHK, 1, DQK)
    q, k = (0.995 * t / t.norm(dim=-1, keepdim=True) for t in (q, k))  # below 1 after rounding to 8 bits
    v = n(B, NH, S, DV)
    g = -torch.exp(-5 * torch.rand(B, NH, 1, generator=r)) * torch.nn.functional.softplus(n(B, NH, S)) * (20 if strong else 1)
    beta = torch.sigmoid(n(B, NH, S))
    c0 = 0.5 * n(B, NH, DQK, DV) if state else None
    to = lambda t, d: t.to(d).to(device)  # noqa: E731
    return to(q, dtype), to(k, dtype), to(v, dtype), to(g, gate), to(beta, gate), None if c0 is None else c0.to(device)


def reference(q, k, v, g, beta, c0, ku, scale=None, planes=False, chunk=None):
    """h, C in float64 and their bars (h's without its own rounding); planes: h's operands are single f16 planes;
    chunk: the chunkwise kernels' tokens of a chunk (by default where ku is theirs)."""
    q, k, v, g, beta = (t.double() for t in (q, k, v, g, beta))
    B, NH, S, DV = v.shape
    DQK, rep = q.shape[-1], NH // q.shape[1]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    scale = DQK ** -0.5 if scale is None else scale
    C = torch.zeros(B, NH, DQK, DV, dtype=torch.float64, device=v.device) if c0 is None else c0.double()
    E, floor = ku * C.norm(dim=-2), 0.0
    a = torch.exp(g)
    chunk = 64 if chunk is None and ku >= CHUNK_KU else chunk
    h, bar, U, top = torch.empty_like(v), torch.empty_like(v), torch.empty_like(v), C.norm(dim=-2)
    for t in range(S):
        kt, at = k[:, :, t], a[:, :, t, None]
        if chunk and t % chunk == 0:
            floor = 2.0 ** -34 * C.norm(dim=-2).amax(-1, keepdim=True)
        start = C.norm(dim=-2) * at if chunk and t % chunk == 0 else start * at if chunk else 0 * E
        C = C * at[..., None]
        U[:, :, t] = beta[:, :, t, None] * (v[:, :, t] - (kt[..., None] * C).sum(-2))
        C = C + kt[..., None] * U[:, :, t, None, :]
        size = torch.maximum(C.norm(dim=-2), start)
        top = torch.maximum(top, size)
        E = at * E + floor + ku * (size + U[:, :, t].abs() * kt.norm(dim=-1, keepdim=True) + beta[:, :, t, None] * v[:, :, t].abs())
        h[:, :, t] = scale * (q[:, :, t, :, None] * C).sum(-2)
        bar[:, :, t] = scale * q[:, :, t].norm(dim=-1, keepdim=True) * (E + ku * size)
    if planes:
        b = g.clamp_min(-1e4).cumsum(-1)
        low = torch.ones(S, S, dtype=torch.bool, device=v.device).tril()
        D = torch.exp((b[..., :, None] - b[..., None, :]).masked_fill(~low, -torch.inf))
        P = scale * D * (q @ k.transpose(-1, -2)).abs()
        bar = bar + 2.0 ** -11 * (scale * q.norm(dim=-1, keepdim=True) * top[:, :, None] + 2 * P @ U.abs())
    return h, C, bar, E[:, :, None].expand_as(C)


def check(got, want, bar, what):
    from helpers import half_ulp
    # half_ulp is of normal numbers; f16's below 2^-14 are 2^-24 apart, so their rounding is up to 2^-25 off
    ulp = half_ulp(want, got.dtype).clamp_min(2.0 ** -25 if got.dtype == torch.float16 else 0.0).to(want.device)
    err = (got.detach().double() - want).abs() - bar - ulp
    assert got.shape == want.shape and bool((err <= 0).all()), f"{what}: {float(err.max()):.3e} over the bar"
