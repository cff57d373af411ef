"""The gated delta rule on the GPU (chunkwise forward, token by token, decode step) against 64 bits; bars in
delta_reference."""

import pytest
import torch

from delta_reference import CHUNK_KU, check, make, recurrent_ku, reference
from helpers import dev

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

# every padded width, odd ones, columns that fill no wave, one token, chunks' ends, shared heads
SHAPES = [(1, 1, 1, 1, 64, 16), (2, 2, 2, 64, 64, 64), (1, 2, 2, 65, 128, 128), (1, 4, 2, 63, 32, 40), (1, 1, 1, 200, 256, 96),
          (2, 3, 1, 130, 33, 17), (1, 2, 1, 257, 100, 200), (3, 2, 2, 17, 1, 1), (1, 2, 2, 129, 200, 5), (1, 8, 8, 70, 96, 512)]


def chunk_bars(x, **kw):
    return reference(*x, CHUNK_KU, planes=x[0].dtype == BF16, **kw)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype,gate", [(BF16, F32), (BF16, BF16), (F16, F16), (F16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("state", [False, True])
def test_chunkwise(gpu_case, shape, dtype, gate, state):
    import xlstm_hip
    x = make(*shape, dtype, gate, seed=sum(shape), state=state)
    h, c = xlstm_hip.gated_delta_chunkwise(*x, return_last_states=True)
    hr, cr, hb, cb = chunk_bars(x)
    assert h.dtype == dtype and c.dtype == F32
    check(c, cr, cb, "C")
    check(h, hr, hb, "h")
    assert torch.equal(h, xlstm_hip.gated_delta_chunkwise(*x))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype,gate", [(BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("state", [False, True])
def test_recurrent(gpu_case, shape, dtype, gate, state):
    import xlstm_hip
    x = make(*shape, dtype, gate, seed=sum(shape) + 1, state=state)
    h, c = xlstm_hip.gated_delta_recurrent(*x, return_last_states=True)
    hr, cr, hb, cb = reference(*x, recurrent_ku(shape[4]))
    check(c, cr, cb, "C")
    check(h, hr, hb, "h")
    assert torch.equal(h, xlstm_hip.gated_delta_recurrent(*x))


@pytest.mark.parametrize("shape", [(64, 8, 4, 11, 100, 50), (40, 8, 8, 3, 256, 64), (32, 16, 16, 17, 33, 33), (8, 33, 11, 8, 64, 31)])
@pytest.mark.parametrize("dtype,gate", [(BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("state", [False, True])
def test_recurrent_of_many_heads(gpu_case, shape, dtype, gate, state):
    test_recurrent(gpu_case, shape, dtype, gate, state)


@pytest.mark.parametrize("B,NH,NHK,DQK,DV", [(1, 8, 8, 128, 256), (5, 4, 2, 64, 40), (3, 3, 1, 33, 7), (16, 8, 8, 256, 512)])
@pytest.mark.parametrize("dtype,gate", [(BF16, BF16), (F16, F32), (F32, F32)])
def test_step(gpu_case, B, NH, NHK, DQK, DV, dtype, gate):
    import xlstm_hip
    x = make(B, NH, NHK, 1, DQK, DV, dtype, gate, seed=B + DQK)
    hr, cr, hb, cb = reference(*x, recurrent_ku(DQK))
    one = [t[:, :, 0] for t in x[:5]]
    kept = x[5].clone()
    h, c = xlstm_hip.gated_delta_step(*one, x[5])
    assert torch.equal(x[5], kept)
    check(h, hr[:, :, 0], hb[:, :, 0], "h")
    check(c, cr, cb, "C")
    h2, c2 = xlstm_hip.gated_delta_step_(*one, x[5])
    assert c2 is x[5] and torch.equal(h, h2) and torch.equal(c, c2)


# many heads: the decode step's own kernels, by their widths, rows and ragged columns
@pytest.mark.parametrize("B,NH,NHK,DQK,DV", [(32, 8, 8, 128, 256), (64, 8, 4, 256, 512), (32, 8, 8, 100, 256), (64, 4, 1, 64, 64),
                                             (40, 8, 8, 33, 100), (64, 4, 4, 200, 196), (64, 4, 4, 1, 4)])
@pytest.mark.parametrize("dtype,gate", [(BF16, F32), (F16, F16), (F32, F32)])
def test_step_of_many_heads(gpu_case, B, NH, NHK, DQK, DV, dtype, gate):
    test_step(gpu_case, B, NH, NHK, DQK, DV, dtype, gate)


# many blocks of columns: the scans' form of one wave a block
MANY = [(32, 8, 8, 70, 64, 64), (16, 8, 4, 130, 128, 100), (32, 8, 8, 65, 256, 40), (8, 16, 16, 64, 200, 128)]


@pytest.mark.parametrize("shape", MANY)
@pytest.mark.parametrize("dtype,gate", [(BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("state", [False, True])
def test_chunkwise_of_many_heads(gpu_case, shape, dtype, gate, state):
    test_chunkwise(gpu_case, shape, dtype, gate, state)


@pytest.mark.parametrize("B,NH,DK,DV", [(2, 128, 100, 256), (1, 3, 70, 33), (1, 2, 1, 1), (3, 100, 256, 255), (1, 5, 129, 66)])
def test_step_of_any_columns(gpu_case, B, NH, DK, DV):
    """One token from a state: columns that nothing divides, the wide kernel's too, also where the state's address is odd."""
    import xlstm_hip
    x = make(B, NH, NH, 1, DK, DV, BF16, F32, seed=DK + DV)
    one = [t[:, :, 0] for t in x[:5]]
    h, c = xlstm_hip.gated_delta_step(*one, x[5])
    hr, cr, hb, cb = reference(*x, recurrent_ku(DK))
    check(c, cr, cb, "C")
    check(h[:, :, None], hr, hb, "h")
    held = torch.full((x[5].numel() + 2,), 7.0, device=dev())
    odd = held[1:-1].view(x[5].shape)
    odd.copy_(x[5])
    h2, _ = xlstm_hip.gated_delta_step_(*one, odd)
    assert torch.equal(h, h2) and torch.equal(odd, c) and float(held[0]) == float(held[-1]) == 7.0
    assert torch.equal(xlstm_hip.gated_delta_recurrent(*x)[:, :, 0], h)


def test_step_on_an_odd_address(gpu_case):
    import xlstm_hip
    x = make(2, 2, 2, 1, 64, 32, BF16, BF16, seed=3)
    one = [t[:, :, 0] for t in x[:5]]
    want = xlstm_hip.gated_delta_step(*one, x[5])
    held = torch.zeros(x[5].numel() + 1, device=dev())
    c = held[1:].view(x[5].shape)
    c.copy_(x[5])
    h, _ = xlstm_hip.gated_delta_step_(*one, c)
    assert torch.equal(h, want[0]) and torch.equal(c, want[1]) and float(held[0]) == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_long_and_in_pieces(gpu_case, dtype):
    """Thousands of tokens; the state carried from piece to piece; prefill, then drafted tokens, then steps."""
    import xlstm_hip
    x = make(1, 2, 2, 3001, 64, 48, dtype, F32, seed=5)
    hr, cr, hb, cb = reference(*x, 2 * CHUNK_KU)
    if dtype == BF16:
        hb = hb + 2.0 ** -9 * hr.abs().max()
    h, c = xlstm_hip.gated_delta_chunkwise(*x, return_last_states=True)
    check(h, hr, hb, "h")
    check(c, cr, cb, "C")
    c, at = x[5], 0
    for n in (1000, 77, 1900, 20):
        part = [t[:, :, at:at + n] for t in x[:5]]
        op = xlstm_hip.gated_delta_recurrent if n < 64 else xlstm_hip.gated_delta_chunkwise
        h, c = op(*part, c, return_last_states=True)
        check(h, hr[:, :, at:at + n], hb[:, :, at:at + n], f"h from {at}")
        at += n
    for t in range(at, 3001):
        h, c = xlstm_hip.gated_delta_step_(*(y[:, :, t] for y in x[:5]), c)
        check(h, hr[:, :, t], hb[:, :, t], f"h of {t}")
    check(c, cr, cb, "C after the pieces")


@pytest.mark.parametrize("op", ["gated_delta_chunkwise", "gated_delta_recurrent"])
def test_no_tokens(gpu_case, op):
    import xlstm_hip
    x = make(2, 2, 1, 3, 64, 40, BF16, F32, seed=1)
    none = [t[:, :, :0] for t in x[:5]]
    h, c = getattr(xlstm_hip, op)(*none, x[5], return_last_states=True)
    assert h.shape == (2, 2, 0, 40) and torch.equal(c, x[5])
    _, c = getattr(xlstm_hip, op)(*none, return_last_states=True)
    assert c.shape == x[5].shape and float(c.abs().max()) == 0


@pytest.mark.parametrize("op,ku", [("gated_delta_chunkwise", CHUNK_KU), ("gated_delta_recurrent", recurrent_ku(64))])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_resets_and_padding(gpu_case, op, ku, dtype):
    """g = -inf starts afresh (several in one chunk); strong decays; tokens with g and beta 0 leave the state alone."""
    import xlstm_hip
    q, k, v, g, beta, c0 = make(1, 2, 2, 150, 64, 48, dtype, F32, seed=9, strong=True)
    for t in (0, 5, 6, 40, 64, 127, 128, 149):
        g[:, :, t] = -torch.inf
    g[:, :, 70:100] = 0
    beta[:, :, 70:100] = 0
    x = (q, k, v, g, beta, c0)
    planes = dtype == BF16 and op == "gated_delta_chunkwise"
    hr, cr, hb, cb = reference(*x, ku, planes=planes)
    h, c = getattr(xlstm_hip, op)(*x, return_last_states=True)
    check(h, hr, hb, "h")
    check(c, cr, cb, "C")
    # what is before a reset leaves no trace at all
    _, c1 = getattr(xlstm_hip, op)(*(t[:, :, 128:] for t in x[:5]), None, return_last_states=True)
    check(c1, cr, cb, "C from the reset on")


@pytest.mark.parametrize("ks,vs,cs", [(1e-6, 1.0, 1.0), (1.0, 1e6, 1e6), (1.0, 1e-6, 1e-6), (1e-3, 1e-12, 0.0), (1.0, 1.0, 1e20)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_ranges(gpu_case, ks, vs, cs, dtype):
    """Values far from 1: every operand is scaled into f16's range."""
    import xlstm_hip
    q, k, v, g, beta, c0 = make(1, 2, 2, 140, 64, 48, F32, F32, seed=11)
    x = ((q * 3e4).to(dtype), (k * ks).to(dtype), (v * vs).to(dtype), g, beta, c0 * cs)
    hr, cr, hb, cb = reference(*x, CHUNK_KU, planes=dtype == BF16)
    h, c = xlstm_hip.gated_delta_chunkwise(*x, return_last_states=True)
    check(h, hr, hb, "h")
    check(c, cr, cb, "C")


def test_zeros(gpu_case):
    import xlstm_hip
    x = make(1, 2, 2, 100, 64, 48, BF16, BF16, seed=2)
    for i in range(3):
        y = list(x)
        y[i] = torch.zeros_like(y[i])
        hr, cr, hb, cb = reference(*y, CHUNK_KU, planes=True)
        h, c = xlstm_hip.gated_delta_chunkwise(*y, return_last_states=True)
        check(h, hr, hb, "h")
        check(c, cr, cb, "C")
    h, c = xlstm_hip.gated_delta_chunkwise(*(torch.zeros_like(t) for t in x[:5]), return_last_states=True)
    assert float(h.abs().max()) == 0 and float(c.abs().max()) == 0


def test_equal_keys(gpu_case):
    """The same key at every token, beta 1: T's entries do not decay; the state answers the last value."""
    import xlstm_hip
    q, k, v, g, beta, _ = make(1, 1, 1, 150, 64, 32, F32, F32, seed=4)
    k = k[:, :, :1].expand_as(k).contiguous()
    x = (k, k, v, torch.zeros_like(g), torch.ones_like(beta), None)
    hr, cr, hb, cb = reference(*x, CHUNK_KU)
    h, c = xlstm_hip.gated_delta_chunkwise(*x, return_last_states=True)
    check(h, hr, hb, "h")
    check(c, cr, cb, "C")


def test_not_finite_stays_in_its_chunk(gpu_case):
    import xlstm_hip
    x = make(1, 2, 2, 200, 64, 48, BF16, F32, seed=6)
    want = xlstm_hip.gated_delta_chunkwise(*x)
    for i in (0, 1, 2):
        y = [t.clone() for t in x]
        y[i][0, 1, 130] = float("nan")
        h = xlstm_hip.gated_delta_chunkwise(*y)
        assert torch.equal(h[:, 0], want[:, 0]) and torch.equal(h[:, 1, :128], want[:, 1, :128])
        assert bool(torch.isnan(h[0, 1, 130:131]).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides(gpu_case, dtype):
    """A projection's transposed views, slices of wider rows, odd offsets, expanded heads, gates of other strides."""
    import xlstm_hip
    x = make(2, 4, 4, 90, 64, 48, dtype, F32, seed=8)
    want = xlstm_hip.gated_delta_chunkwise(*x, return_last_states=True)

    def lay(t, kind):
        if kind == "transposed":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if kind == "wide":
            w = torch.full(t.shape[:-1] + (t.shape[-1] + 13,), 7.0, dtype=t.dtype, device=t.device)
            w[..., 5:5 + t.shape[-1]] = t
            return w[..., 5:5 + t.shape[-1]]
        if kind == "columns apart":
            return t.transpose(2, 3).contiguous().transpose(2, 3)
        w = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        w[1:] = t.reshape(-1)
        return w[1:].view(t.shape)

    for kind in ("transposed", "wide", "columns apart", "odd start"):
        y = [lay(t, kind) for t in x[:3]] + [t.transpose(1, 2).contiguous().transpose(1, 2) for t in x[3:5]] + [x[5]]
        assert all(torch.equal(a, b) for a, b in zip(y, x))
        for op in (xlstm_hip.gated_delta_chunkwise, xlstm_hip.gated_delta_recurrent):
            got = op(*y, return_last_states=True)
            plain = want if op is xlstm_hip.gated_delta_chunkwise else op(*x, return_last_states=True)
            assert all(torch.equal(a, b) for a, b in zip(got, plain)), kind
    q1 = x[0][:, :1].expand_as(x[0])
    assert torch.equal(xlstm_hip.gated_delta_chunkwise(q1, *x[1:]), xlstm_hip.gated_delta_chunkwise(q1.contiguous(), *x[1:]))


def test_scale(gpu_case):
    import xlstm_hip
    x = make(1, 2, 2, 80, 64, 48, F32, F32, seed=12)
    for scale in (0.0, 1.0, -2.5):
        hr, _, hb, _ = reference(*x, CHUNK_KU, scale=scale)
        check(xlstm_hip.gated_delta_chunkwise(*x, scale=scale), hr, hb.abs(), "h")
        check(xlstm_hip.gated_delta_recurrent(*x, scale=scale), hr, hb.abs(), "h")


def test_other_stream(gpu_case):
    import xlstm_hip
    x = make(2, 2, 2, 500, 64, 64, BF16, F32, seed=13)
    want = xlstm_hip.gated_delta_chunkwise(*x, return_last_states=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(xlstm_hip.gated_delta_chunkwise(*x, return_last_states=True))
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, want))
