"""The gated delta rule on the GPU where sizes are far apart: gradients beside a matrix of zeros, keys far below 1, rows of one chunk
far from each other, columns that are not finite.

Bars of gradients are those of test_gpu_gated_delta_bwd, of a head or (``token_parts``) of each token's own terms; of h and the state
delta_reference's, but that what a token adds to the state is taken at its key's length (``tight``)."""

import pytest
import torch

from delta_reference import CHUNK_KU, check, make, reference
from helpers import dev
from test_gpu_gated_delta_bwd import BAR, check_all, gradients, inputs, plain

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


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


# ------------------------------------------------------------------ rows of one chunk far apart
def row_sizes(kind, S):
    """(of q's rows, of k's): a token's own size."""
    one, t = torch.ones(S), torch.arange(S)
    far = 10.0 ** -(6.0 * torch.rand(S, generator=torch.Generator().manual_seed(S)))
    small = torch.where(t % 5 == 2, 1e-6, 1.0)
    # keys that grow in the middle of a chunk: those before it are small beside their chunk's largest
    early = torch.where(t < 40, 1e-6, 1.0)
    return {"q": (far, one), "q small": (small, one), "k early": (one, early), "k late": (one, early.flip(0)), "both": (far.flip(0), far)}[kind]


KINDS = ["q", "q small", "k early", "k late", "both"]


@pytest.mark.parametrize("shape", [(1, 2, 2, 140, 64, 48), (1, 2, 1, 100, 200, 40), (40, 8, 8, 70, 128, 20)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("state", [False, True])
def test_rows_far_apart(gpu_case, shape, dtype, kind, state):
    """h of every token to its own size, whatever the other tokens' queries and keys are."""
    import xlstm_hip
    if dtype == F16:  # its own numbers end at 2^-24: rows of 1e-3 at the least, and h on a scale that its numbers hold
        sizes = [s.clamp_min(1e-3) for s in row_sizes(kind, shape[3])]
    else:
        sizes = row_sizes(kind, shape[3])
    q, k, v, g, beta, c0 = make(*shape, F32, F32, seed=41, state=state)
    q, k = (t * s.to(dev())[:, None] for t, s in zip((q, k), sizes))
    x = (q.to(dtype), k.to(dtype), v.to(dtype), g, beta, c0)
    hr, cr, hb, cb = tight(*x, planes=dtype == BF16)
    h, c = xlstm_hip.gated_delta_chunkwise(*x, return_last_states=True)
    check(c, cr, cb, "C")
    check(h, hr, hb, "h")


def token_parts(x, dh, scale):
    """Sizes of a token's dq, dk and dv before anything cancels, without an initial or last state: norms of the sums' terms."""
    q, k, v, g, beta = (t.double() for t in x[:5])
    rep = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    C, U, Gs = v.new_zeros(*v.shape[:2], q.shape[-1], v.shape[-1]), torch.empty_like(v), torch.empty_like(v)
    for t in range(v.shape[2]):
        C = C * torch.exp(g[:, :, t, None, None])
        U[:, :, t] = beta[:, :, t, None] * (v[:, :, t] - (k[:, :, t, :, None] * C).sum(-2))
        C = C + k[:, :, t, :, None] * U[:, :, t, None, :]
    G = torch.zeros_like(C)
    for t in reversed(range(v.shape[2])):
        G = G + scale * q[:, :, t, :, None] * dh.double()[:, :, t, None, :]
        Gs[:, :, t] = (k[:, :, t, :, None] * G).sum(-2)  # dU = Z
        G = torch.exp(g[:, :, t, None, None]) * (G - k[:, :, t, :, None] * (beta[:, :, t, None] * Gs[:, :, t])[..., None, :])
    b = g.cumsum(-1)
    low = torch.ones(g.shape[-1], g.shape[-1], dtype=torch.bool, device=g.device).tril()
    D = torch.exp((b[..., :, None] - b[..., None, :]).masked_fill(~low, -torch.inf))
    n = lambda t: t.norm(dim=-1)  # noqa: E731
    lq, lk, ld, lu, lz = n(q), n(k), n(dh.double()), n(U), n(Gs)
    M = D * low.double().tril(-1)
    dq = scale * (D * ld[..., :, None] * lu[..., None, :] @ lk[..., None])[..., 0]
    dk = scale * ((D * ld[..., :, None] * lu[..., None, :]).mT @ lq[..., None])[..., 0]
    E = M * (beta * lz)[..., :, None] * lu[..., None, :]
    dk = dk + ((E + E.mT) @ lk[..., None])[..., 0]
    dv = scale * ((D * lq[..., :, None] * lk[..., None, :]).mT @ ld[..., None])[..., 0]
    dv = beta * (lz + dv + lk * (M.mT @ (beta * lz * lk)[..., None])[..., 0])
    share = lambda t: t.view(t.shape[0], -1, rep, t.shape[-1]).sum(2)  # noqa: E731
    return share(dq), share(dk), dv


@pytest.mark.parametrize("shape", [(1, 2, 2, 140, 64, 48), (1, 2, 1, 100, 200, 40), (16, 8, 8, 70, 128, 48)])
@pytest.mark.parametrize("kind", KINDS)
def test_gradients_of_rows_far_apart(gpu_case, shape, kind):
    """dq, dk and dv of every token to the size of its own terms, float32: 10 pairs' roundings of 2^-22 (test_gpu_gated_delta_bwd's
    count, twice).  Queries and keys have rows 2^-20 of the largest, so products of both have 2^-40.  The operands that are formed of such
    (dU, Z, and what K and Q are multiplied with for dQ and dK) stand at 2^14 of their block or chunk and f16 ends at 2^-24: each value
    is off by 2^-39 of the largest, and 64 of them, of random sign, with factors up to 1, by sqrt(64) of that, with two or three operands one behind the
    other by 2^-34 of the largest token's."""
    import xlstm_hip
    x, dh, _ = inputs(shape, F32, F32, 43, state=False, last=False)
    x = [t * s.to(dev())[:, None] for t, s in zip(x[:2], row_sizes(kind, shape[3]))] + list(x[2:])
    scale = shape[4] ** -0.5
    got = gradients(lambda *y: (xlstm_hip.gated_delta_chunkwise(*y, scale=scale), None), x, dh, None)
    want = gradients(lambda *y: plain(*y, scale), x, dh, None, torch.float64)
    for a, w, part, name in zip(got, want, token_parts(x, dh, scale), ("dq", "dk", "dv")):
        err = (a.double() - w).norm(dim=-1)
        largest = torch.cat([c.amax(-1, keepdim=True).expand_as(c) for c in part.split(64, -1)], -1)
        worst = float(((err - 2.0 ** -34 * largest) / part.clamp_min(1e-300)).max())
        assert worst <= BAR[F32], f"{name}: {worst:.3e} of a token's terms"


# ------------------------------------------------------------------ columns that are not finite
@pytest.mark.parametrize("shape", [(1, 2, 2, 200, 64, 48), (1, 1, 1, 140, 256, 40), (40, 8, 8, 140, 64, 20)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("size", [1.0, 1e7, 1e-7])
def test_not_finite_stays_in_its_column(gpu_case, shape, dtype, value, size):
    """One value of v, or of the state, that is not finite: the 15 columns beside it keep their results, and so does
    what its own column had in earlier chunks."""
    import xlstm_hip
    x = list(make(*shape, F32, F32, seed=51))
    x[2], x[5] = x[2] * size, x[5] * size
    x[:3] = (t.to(dtype) for t in x[:3])
    hr, cr, hb, cb = reference(*x, CHUNK_KU, planes=dtype == BF16)
    others = torch.arange(shape[5], device=dev()) != 3
    for where in ("v", "c"):
        y = [t.clone() for t in x]
        if where == "v":
            y[2][0, -1, 130, 3] = value
        else:
            y[5][0, -1, 5, 3] = value
        h, c = xlstm_hip.gated_delta_chunkwise(*y, return_last_states=True)
        check(h[..., others], hr[..., others], hb[..., others], f"h, {where}")
        check(c[..., others], cr[..., others], cb[..., others], f"C, {where}")
        check(h[:, :-1], hr[:, :-1], hb[:, :-1], f"h of other heads, {where}")
        if where == "v":
            check(h[:, :, :128], hr[:, :, :128], hb[:, :, :128], "h of earlier chunks")


@pytest.mark.parametrize("shape", [(1, 2, 2, 100, 64, 48), (16, 8, 8, 70, 128, 48)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_beside_a_column_that_is_not_finite(gpu_case, shape, dtype):
    """dH of one column is infinite: dv and dc0 of the other columns are what they were (dq, dk and the gates' sum over all of them)."""
    import xlstm_hip
    (q, k, v, g, beta, c0), dh, dc = inputs(shape, dtype, F32, 52)
    x, dh, dc = (q, k, v, g, beta, c0), dh * 1e6, dc * 1e6
    fn = lambda *y: xlstm_hip.gated_delta_chunkwise(*y, return_last_states=True)  # noqa: E731
    want = gradients(lambda *y: plain(*y, shape[4] ** -0.5), x, dh, dc, torch.float64)
    spoilt = dh.clone()
    spoilt[:, :, 37, 3] = float("inf")
    got = gradients(fn, x, spoilt, dc)
    others = torch.arange(shape[5], device=dev()) != 3
    for i in (2, 5):
        a, w = (t[..., others].double().flatten(2) for t in (got[i], want[i]))
        worst = float(((a - w).norm(dim=-1) / w.norm(dim=-1)).max())
        assert worst <= BAR[dtype] + torch.finfo(got[i].dtype).eps / 2, f"{i}: {worst:.3e}"


@pytest.mark.parametrize("shape", [(1, 2, 2, 140, 64, 48), (40, 8, 8, 70, 64, 20)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_rows_of_zeros(gpu_case, shape, dtype, which):
    """Tokens whose q, k or v is zeros, alone and a chunk of them, beside others: their h, and dk or dq, which do not vanish."""
    import xlstm_hip
    x, dh, dc = inputs(shape, dtype, F32, 61)
    x[which][:, :, 3:9] = 0
    x[which][:, :, -1] = 0
    x[which][:, :, 64:] = 0
    hr, cr, hb, cb = tight(*x, planes=dtype == BF16)
    h, c = xlstm_hip.gated_delta_chunkwise(*x, return_last_states=True)
    check(c, cr, cb, "C")
    check(h, hr, hb, "h")
    if shape[0] == 1:
        check_all(x, dh, dc)


# ------------------------------------------------------------------ small writes into a large state
@pytest.mark.parametrize("shape", [(1, 2, 2, 2560, 64, 48), (1, 1, 1, 1920, 256, 32), (1, 2, 2, 1280, 128, 64), (40, 8, 8, 640, 64, 20)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("by", ["beta", "k"])
def test_small_writes_add_up(gpu_case, shape, dtype, by):
    """Tokens that each write 1e-6 or less of the state, without decay (gates all but closed, or short keys): thousands of them are seen.

    Bar, of the largest value of the state (a column's block has one scale): a chunk rounds the state to float32 and takes its writes
    at 2^-31 of it, 64 of them: 2^-22 in all; a write is off by 16 2^-22 of itself (delta_reference)."""
    import xlstm_hip
    B, NH, _, S, DQK, DV = shape
    r = torch.Generator().manual_seed(71)
    unit = torch.nn.functional.normalize(torch.randn(B, NH, 1, DQK, generator=r), dim=-1).expand(B, NH, S, DQK)
    v = torch.rand(B, NH, S, DV, generator=r) + 0.5
    size = {"beta": (1e-6, 1.0), "k": (0.7, 2.0 ** -20)}[by]
    q, k, v = unit.to(dtype).to(dev()), (unit * size[1]).to(dtype).to(dev()), v.to(dtype).to(dev())
    g, beta = torch.zeros(B, NH, S, device=dev()), torch.full((B, NH, S), size[0], device=dev())
    # a state that does not answer to the keys: every token writes beta v
    c0 = torch.randn(B, NH, DQK, DV, generator=r).to(dev())
    u = k[:, :, 0].double() / k[:, :, 0].double().norm(dim=-1, keepdim=True)
    c0 = (c0.double() - u[..., None] * (u[..., None] * c0.double()).sum(-2, keepdim=True)).float()
    want = c0.double()
    kd, vd, bd = k[:, :, 0].double(), v.double(), float(beta[0, 0, 0].double())
    # k is the same at every token: C's part along it goes to x - beta |k|^2 x + beta v by itself
    along, n2 = (kd[..., None] * want).sum(-2), (kd ** 2).sum(-1)[..., None]
    total = torch.zeros_like(along)
    for t in range(S):
        d = bd * (vd[:, :, t] - along)
        along, total = along + n2 * d, total + d
    want = want + kd[..., None] * total[..., None, :]
    _, c = xlstm_hip.gated_delta_chunkwise(q, k, v, g, beta, c0, return_last_states=True)
    chunks = (S + 63) // 64
    bar = chunks * 2.0 ** -22 * float(want.abs().max()) + CHUNK_KU * float((kd[..., None] * total[..., None, :]).abs().max())
    err = float((c.double() - want).abs().max())
    assert err <= bar, f"{err:.3e} over {bar:.3e}; written {float((want - c0).abs().max()):.3e}"


@pytest.mark.parametrize("shape", [(1, 2, 2, 200, 64, 48), (1, 1, 1, 200, 256, 32), (40, 8, 8, 140, 128, 20)])
@pytest.mark.parametrize("size", [1e6, 1e8])
def test_large_values_at_short_keys(gpu_case, shape, size):
    """A token in 16 whose v is 1e6 (1e8) times the others' and whose k as much shorter: its U is large, what it writes is not, and the state and
    the other tokens' writes keep their bits, float32.

    Bar: 16 2^-22 of the state's columns and of the chunk's writes (delta_reference), at q's length; and U is off by 2^-39 of its block's
    largest: of a state of 64 tokens' (random signs) 2^-36 of it, twice that where a chunk's products take it again."""
    import xlstm_hip
    q, k, v, g, beta, _ = make(*shape, F32, F32, seed=81, state=False)
    rare = (torch.arange(shape[3], device=dev()) % 16 == 5)[:, None]
    k, v = torch.where(rare, k / size, k), torch.where(rare, v * size, v)
    hr, cr, hb, cb = tight(q, k, v, g, beta, None)
    B, NH, S = g.shape
    kd, scale = k.double().repeat_interleave(NH // k.shape[1], 1), shape[4] ** -0.5
    C, bar, writes = torch.zeros_like(cr), torch.empty_like(hr), 0.0
    lq = q.double().norm(dim=-1).repeat_interleave(NH // k.shape[1], 1)
    most, largest = 0.0, float(v.abs().max())
    for t in range(S):
        C = C * torch.exp(g[:, :, t].double())[..., None, None]
        d = beta[:, :, t, None].double() * (v[:, :, t].double() - (kd[:, :, t, :, None] * C).sum(-2))
        C = C + kd[:, :, t, :, None] * d[..., None, :]
        most = torch.maximum(torch.as_tensor(most, device=dev()), C.norm(dim=-2))
        writes = writes + (kd[:, :, t].norm(dim=-1, keepdim=True) * d).abs()
        bar[:, :, t] = scale * lq[:, :, t, None] * (CHUNK_KU * (most + writes) + 2.0 ** -35 * largest)
    h, c = xlstm_hip.gated_delta_chunkwise(q, k, v, g, beta, return_last_states=True)
    err = (h.double() - hr).abs() / bar
    assert float(err.max()) <= 1, f"h: {float(err.max()):.2f} of the bar"


# ------------------------------------------------------------------ padding
@pytest.mark.parametrize("shape", [(1, 2, 2, 150, 64, 48), (1, 2, 1, 100, 200, 40), (40, 8, 8, 140, 64, 20)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("large", [1.0, 1e9, 1e15])
def test_padding_of_any_values(gpu_case, shape, dtype, large):
    """Tokens of g and beta 0, scattered and a run over a chunk's border, with whatever is in their q, k and v: the others' h and the state are
    those of the sequence without them."""
    import xlstm_hip
    x = make(*shape, dtype, F32, seed=91)
    S = shape[3]
    t = torch.arange(S)
    pad = (t % 7 == 3) | ((t > 50) & (t < 75))
    y = [a.clone() for a in x]
    y[3][:, :, pad], y[4][:, :, pad] = 0, 0
    keep = (~pad).to(dev())
    hr, cr, hb, cb = reference(*[a[:, :, keep] for a in y[:5]], y[5], CHUNK_KU, planes=dtype == BF16)
    for i in range(3):
        y[i][:, :, pad] *= large
    h, c = xlstm_hip.gated_delta_chunkwise(*y, return_last_states=True)
    # chunks are cut where they would not be without the padding: a second chunk's start as large as the first's
    check(c, cr, 2 * cb, "C")
    check(h[:, :, keep], hr, 2 * hb, "h")
