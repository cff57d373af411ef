"""Gradients of the gated delta rule on the GPU to the bits of their own types: float32 ones (the gates', a carried state's) of 16-bit
inputs, and all of float16's.

Bars: the backward's operands are pairs of f16 there, so each gradient is off by test_gpu_gated_delta_bwd's count for float32 (10 roundings of 2^-22 +
4.5 2^-24, two parts: BAR[F32]) of the norm of its terms, and by its own rounding.  dq, dk, dv and dc0 are compared by head and
norm; a gate's gradient by head with the norm of its own terms (``gate_parts``): a sum of rounded products x y is off by the rounding
times sqrt(sum x^2 y^2), roundings being unrelated."""

import pytest
import torch

from test_gpu_gated_delta_bwd import BAR, NAMES, SHAPES, direct_part, gradients, inputs, plain

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gate_parts(x, dh, dc, scale):
    """Norms of the terms of (dg, dbeta) at every token, by chunks of 64 (csrc/delta_backward.hip has the formulas)."""
    q, k, v, g, beta = (t.double() for t in x[:5])
    rep = v.shape[1] // q.shape[1]
    q, k, dh = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1), dh.double()
    S, a = v.shape[2], torch.exp(g)
    C = v.new_zeros(*v.shape[:2], q.shape[-1], v.shape[-1]) if x[5] is None else x[5].double()
    U, Z, before, behind = torch.empty_like(v), torch.empty_like(v), [], []
    for t in range(S):
        if t % 64 == 0:
            before.append(C)
        C = C * a[:, :, t, None, None]
        U[:, :, t] = beta[:, :, t, None] * (v[:, :, t] - (k[:, :, t, :, None] * C).sum(-2))
        C = C + k[:, :, t, :, None] * U[:, :, t, None, :]
    G = torch.zeros_like(C) if dc is None else dc.double()
    for t in reversed(range(S)):
        if t % 64 == 63 or t == S - 1:
            behind.insert(0, G)
        G = G + scale * q[:, :, t, :, None] * dh[:, :, t, None, :]
        Z[:, :, t] = (k[:, :, t, :, None] * G).sum(-2)
        G = a[:, :, t, None, None] * (G - k[:, :, t, :, None] * (beta[:, :, t, None] * Z[:, :, t])[..., None, :])
    dg, db = torch.empty_like(g), torch.empty_like(g)
    for c, (S0, dS) in enumerate(zip(before, behind)):
        at = slice(64 * c, min(S, 64 * c + 64))
        qc, kc, vc, uc, zc, hc, bc = (t[:, :, at] for t in (q, k, v, U, Z, dh, beta))
        b = g[:, :, at].cumsum(-1)
        low = torch.ones(b.shape[-1], b.shape[-1], dtype=torch.bool, device=b.device).tril()
        D = torch.exp((b[..., :, None] - b[..., None, :]).masked_fill(~low, -torch.inf))
        c_in, c_out = torch.exp(b), torch.exp(b[..., -1:] - b)
        P, N = scale * D * (qc @ kc.mT), (D * (kc @ kc.mT)).tril(-1)
        dP, dA = (hc ** 2 @ uc.mT ** 2), (zc ** 2 @ uc.mT ** 2)  # squares of the terms' norms
        state = lambda r, s, w: ((r ** 2 @ s ** 2) * w ** 2).sum(-1)  # noqa: E731
        kz, qs, ks = state(kc, S0, zc) * c_in ** 2, state(qc, S0, hc) * (scale * c_in) ** 2, state(kc, dS, uc) * c_out ** 2
        pair = P ** 2 * dP + bc[..., None] ** 2 * N ** 2 * dA
        terms = pair.sum(-1) + pair.sum(-2) + bc ** 2 * kz + qs + ks
        terms[..., -1] += ks.sum(-1) + torch.exp(b[..., -1]) ** 2 * (S0 ** 2 * dS ** 2).sum((-2, -1))
        dg[:, :, at] = terms.flip(-1).cumsum(-1).flip(-1).sqrt()
        db[:, :, at] = ((zc ** 2 * vc ** 2).sum(-1) + kz + (N ** 2 * dA).sum(-1)).sqrt()
    return dg, db


def check_bits(shape, dtype, gate, seed, state):
    import xlstm_hip
    x, dh, dc = inputs(shape, dtype, gate, seed, state, state)
    scale = shape[4] ** -0.5
    got = gradients(lambda *y: xlstm_hip.gated_delta_chunkwise(*y, scale=scale, return_last_states=True), x, dh, dc)
    want = gradients(lambda *y: plain(*y, scale), x, dh, dc, torch.float64)
    parts = dict(zip(("dg", "dbeta"), gate_parts(x, dh, dc, scale)))
    direct = direct_part(x, dh, dc, scale)
    for a, w, name in zip(got, want, NAMES):
        if a.dtype == BF16:  # its own rounding hides what is looked for here
            continue
        size = parts.get(name, w).flatten(2).norm(dim=-1)
        if name == "dc0":
            size = torch.maximum(size, direct.flatten(2).norm(dim=-1))
        err = (a.double() - w).flatten(2).norm(dim=-1)
        own = 0 * err if a.dtype == F32 else (w.to(a.dtype).double() - w).flatten(2).norm(dim=-1)
        # a value d from one of the type's numbers, moved by e, is rounded to one at most d + 2 e away
        over = err - own - (1 if a.dtype == F32 else 2) * BAR[F32] * size
        assert bool((over <= 0).all()), f"{name}: {float((err / size.clamp_min(1e-300)).max()):.3e} of its terms, over by {float(over.max()):.3e}"


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("state", [False, True])
def test_float32_gates(gpu_case, shape, dtype, state):
    check_bits(shape, dtype, F32, sum(shape), state)


@pytest.mark.parametrize("shape", [(32, 8, 8, 70, 64, 64), (16, 8, 4, 130, 128, 100), (32, 8, 8, 65, 256, 40)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_float32_gates_of_many_heads(gpu_case, shape, dtype):
    check_bits(shape, dtype, F32, sum(shape), True)


@pytest.mark.parametrize("gate", [BF16, F16])
def test_carried_state(gpu_case, gate):
    """dc0 is float32 whatever the gates are."""
    check_bits((2, 2, 1, 150, 64, 48), BF16, gate, 7, True)


@pytest.mark.parametrize("shape", SHAPES + [(32, 8, 8, 70, 64, 64), (16, 8, 4, 130, 128, 100), (32, 8, 8, 65, 256, 40)])
@pytest.mark.parametrize("state", [False, True])
def test_float16(gpu_case, shape, state):
    """Every gradient of float16 inputs and gates is off by its own rounding: one plane in place of a pair, or one misread, shows."""
    check_bits(shape, F16, F16, sum(shape), state)
