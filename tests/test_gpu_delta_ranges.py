"""The gated delta rule on the GPU where sizes are far apart: gradients beside a matrix of zeros, keys far below 1.

Bars of gradients are those of test_gpu_gated_delta_bwd; of h and the state delta_reference's, but that what a token adds to the state is taken
at its key's length (``tight``)."""

import pytest
import torch

from delta_reference import CHUNK_KU, check, make
from test_gpu_gated_delta_bwd import check_all, inputs

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


# ------------------------------------------------------------------ gradients beside zeros
# one token in the last chunk: there no pair of tokens, and E is zeros; both forms of the scans
@pytest.mark.parametrize("shape", [(1, 2, 2, 1, 64, 48), (1, 2, 2, 65, 64, 48), (1, 2, 1, 129, 100, 40), (16, 8, 8, 65, 128, 48)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vs,ds", [(1e4, 1e4), (1e8, 1e8), (1.0, 1e-12)])
def test_gradients_of_one_token(gpu_case, shape, dtype, vs, ds):
    (q, k, v, g, beta, c0), dh, dc = inputs(shape, dtype, F32, sum(shape))
    check_all((q, k, v * vs, g, beta, c0 * vs), dh * ds, dc * ds)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("what", ["dh", "beta", "v"])
def test_gradients_of_a_chunk_of_zeros(gpu_case, dtype, what):
    """Tokens 64 to 127: no loss, or nothing written, or no values."""
    (q, k, v, g, beta, c0), dh, dc = inputs((1, 2, 2, 180, 64, 48), dtype, F32, 21)
    {"dh": dh, "beta": beta, "v": v}[what][:, :, 64:128] = 0
    check_all((q, k, v * 1e5, g, beta, c0 * 1e5), dh * 1e5, dc * 1e5)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("ks", [1e-6, 1e-12])
def test_gradients_of_small_keys(gpu_case, dtype, ks):
    """The state's gradient against the last state, which every key answers to alone."""
    (q, k, v, g, beta, c0), dh, dc = inputs((1, 2, 2, 65, 64, 48), dtype, F32, 22)
    check_all((q, k * ks, v, g, beta, c0), dh, dc)


# ------------------------------------------------------------------ small keys, blocks of zeros
def tight(q, k, v, g, beta, c0, planes=False):
    """``reference`` with what a token's rounding adds to the state at the length of its key: an error of beta v or of U is
    multiplied by it.  So a state of small keys has as small a bar."""
    q, k, v, g, beta = (t.double() for t in (q, k, v, g, beta))
    B, NH, S, DV = v.shape
    DQK, rep, ku = q.shape[-1], NH // q.shape[1], CHUNK_KU
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    scale, a = DQK ** -0.5, torch.exp(g)
    C = torch.zeros(B, NH, DQK, DV, dtype=torch.float64, device=v.device) if c0 is None else c0.double()
    E, h, bar, U, top = ku * C.norm(dim=-2), torch.empty_like(v), torch.empty_like(v), torch.empty_like(v), torch.empty_like(v)
    most = C.norm(dim=-2)
    for t in range(S):
        kt, at, length = k[:, :, t], a[:, :, t, None], k[:, :, t].norm(dim=-1, keepdim=True)
        if t % 64 == 0:
            floor, start, writes = 2.0 ** -34 * C.norm(dim=-2).amax(-1, keepdim=True), C.norm(dim=-2), 0 * E
            last = min(t + 64, S)
            # U is off by 2^-34 of the largest value that enters its products, of any column
            values = 2.0 ** -34 * (v[:, :, t:last].abs().amax((-2, -1))[..., None] + C.norm(dim=-2).amax(-1, keepdim=True))
        start = start * at
        C = C * at[..., None]
        U[:, :, t] = beta[:, :, t, None] * (v[:, :, t] - (kt[..., None] * C).sum(-2))
        C = C + kt[..., None] * U[:, :, t, None, :]
        # the tokens' parts of the state are rounded at their size, also where they cancel
        writes = writes * at + U[:, :, t].abs() * length
        size = torch.maximum(C.norm(dim=-2), start)
        most = torch.maximum(most, size)
        top[:, :, t] = most
        E = at * E + floor + ku * (size + writes + length * beta[:, :, t, None] * v[:, :, t].abs()) + length * values
        h[:, :, t] = scale * (q[:, :, t, :, None] * C).sum(-2)
        bar[:, :, t] = scale * q[:, :, t].norm(dim=-1, keepdim=True) * (E + ku * (size + writes))
    if planes:
        b = g.clamp_min(-1e4).cumsum(-1)
        low = torch.ones(S, S, dtype=torch.bool, device=v.device).tril()
        D = torch.exp((b[..., :, None] - b[..., None, :]).masked_fill(~low, -torch.inf))
        P = scale * D * (q @ k.transpose(-1, -2)).abs()
        bar = bar + 2.0 ** -11 * (scale * q.norm(dim=-1, keepdim=True) * top + 2 * P @ U.abs())
    return h, C, bar, E[:, :, None].expand_as(C)


# up to 256 blocks of columns: waves share one; more: one a wave
@pytest.mark.parametrize("shape", [(1, 2, 2, 140, 64, 48), (1, 2, 1, 100, 128, 40), (1, 1, 1, 70, 256, 32), (40, 8, 8, 70, 64, 20)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("ks", [1e-9, 1e-20])
@pytest.mark.parametrize("state", [False, True])
def test_small_keys(gpu_case, shape, dtype, ks, state):
    """Ragged last chunks and tokens of beta 0: parts of a chunk whose U is zeros."""
    import xlstm_hip
    q, k, v, g, beta, c0 = make(*shape, F32, F32, seed=31, state=state)
    beta[:, :, 16:52] = 0
    v[..., :16] *= 0 if not state else 1  # zero columns without a state: U is zeros throughout
    x = (q.to(dtype), (k * ks).to(dtype), v.to(dtype), g, beta, c0)
    hr, cr, hb, cb = tight(*x, planes=dtype == BF16)
    h, c = xlstm_hip.gated_delta_chunkwise(*x, return_last_states=True)
    check(c, cr, cb, "C")
    check(h, hr, hb, "h")
