"""Gradients of the gated delta rule on the GPU, against the recurrence's own in 64 bits and against differences.

Bars are of the 2-norm of each gradient of a head.  Every operand of the backward's products is a single f16 plane (bf16, f16: half
a unit, 2^-11) or a pair (float32: 2^-22; and float32 sums), and a gradient passes through a handful of them: the operands of its own product
(2), those of dU, Z and of the state's gradient or U and S before it (at most 8 more).  Roundings are independent, so 10 of them
come to less than 10 units in norm (sqrt(10) if unrelated): 10 x 2^-11 = 4.9e-3 at most in norm for one plane, 10 x (2^-22 + 4.5
2^-24) = 5.1e-6 for pairs, both of the norm of the gradient's largest part.  A gradient is a sum of up to three such parts (dK: with
the states and within the chunk) whose norms may exceed that of their sum by some factor; 2 is allowed for.  For the gates'
gradients, sums of both signs along a chunk, the parts' norm is taken instead: that of dg and dbeta over all heads.  dc0 is the
difference of Q^T dH and K^T Z (decayed), which nearly cancel where the same few keys come again and again (DQK 1: every token halves
the state): the norm of the first, sum_t scale c_t q_t dh_t^T + c_S dc, is taken where it is the larger; the second is at most both together.  To that comes the output's own rounding,
eps / 2 at most."""

import pytest
import torch

from delta_reference import make
from helpers import dev

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
BAR = {F32: 2 * 5.1e-6, BF16: 2 * 4.9e-3, F16: 2 * 4.9e-3}


def plain(q, k, v, g, beta, c0, scale):
    """The recurrence, differentiable, in float64."""
    rep = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    C = v.new_zeros(v.shape[0], v.shape[1], q.shape[-1], v.shape[-1]) if c0 is None else c0
    h = []
    for t in range(v.shape[2]):
        C = C * torch.exp(g[:, :, t, None, None])
        d = beta[:, :, t, None] * (v[:, :, t] - (k[:, :, t, :, None] * C).sum(-2))
        C = C + k[:, :, t, :, None] * d[..., None, :]
        h.append(scale * (q[:, :, t, :, None] * C).sum(-2))
    return torch.stack(h, 2), C


NAMES = ("dq", "dk", "dv", "dg", "dbeta", "dc0")


def gradients(fn, x, dh, dc, dtype=None):
    y = [None if t is None else (t.detach().to(dtype) if dtype else t.detach()).requires_grad_(True) for t in x]
    h, c = fn(*y)
    leaves = [t for t in y if t is not None]
    outs, grads = [], []
    for o, d in ((h, dh), (c, dc)):
        if d is not None:
            outs.append(o)
            grads.append(d.to(o.dtype))
    found = torch.autograd.grad(outs, leaves, grads, allow_unused=True)
    return [torch.zeros_like(t) if f is None else f for f, t in zip(found, leaves)]


def direct_part(x, dh, dc, scale):
    """sum_t scale c_t q_t dh_t^T + c_S dc: the state's gradient before what the tokens' corrections take off."""
    q, g = x[0].double(), x[3].double()
    q = q.repeat_interleave(g.shape[1] // q.shape[1], 1)
    c = torch.exp(g.cumsum(-1))
    part = 0 if dh is None else scale * (q * c[..., None]).transpose(-1, -2) @ dh.double()
    return part if dc is None else part + c[..., -1, None, None] * dc.double()


def compare(got, want, dtype, gate, what="", direct=None):
    for a, w, name in zip(got, want, NAMES):
        assert a.shape == w.shape and bool(torch.isfinite(a).all()), f"{what} {name}"
        bar = BAR[dtype] if dtype != F32 or a.dtype == F32 else BAR[F32]
        rounding = torch.finfo(a.dtype).eps / 2
        if name in ("dg", "dbeta"):
            err, size = (a.double() - w).norm(), w.norm()
        else:
            err, size = (a.double() - w).flatten(2).norm(dim=-1), w.flatten(2).norm(dim=-1)
        if name == "dc0" and direct is not None:
            size = torch.maximum(size, direct.flatten(2).norm(dim=-1))
        worst = float((err / size.clamp_min(1e-300)).max()) if float(size.max()) > 0 else float(err.max())
        assert worst <= bar + rounding, f"{what} {name}: {worst:.3e} of the norm, over {bar + rounding:.3e}"


def inputs(shape, dtype, gate, seed, state=True, last=True, **kw):
    x = make(*shape, dtype, gate, seed=seed, state=state, **kw)
    r = torch.Generator().manual_seed(seed + 1)
    B, NH, _, S, DQK, DV = shape
    dh = torch.randn(B, NH, S, DV, generator=r).to(dtype).to(dev())
    return x, dh, torch.randn(B, NH, DQK, DV, generator=r).to(dev()) if last else None


def check_all(x, dh, dc, scale=None):
    import xlstm_hip
    s = x[0].shape[-1] ** -0.5 if scale is None else scale
    got = gradients(lambda *y: xlstm_hip.gated_delta_chunkwise(*y, scale=scale, return_last_states=True), x, dh, dc)
    want = gradients(lambda *y: plain(*y, s), x, dh, dc, torch.float64)
    for a, t in zip(got, [t for t in x if t is not None]):
        assert a.dtype == t.dtype
    compare(got, want, x[0].dtype, x[3].dtype, direct=direct_part(x, dh, dc, s))
    return got


SHAPES = [(1, 1, 1, 1, 64, 16), (1, 2, 2, 64, 64, 32), (2, 2, 2, 65, 128, 64), (1, 2, 1, 63, 32, 40), (1, 1, 1, 200, 256, 96),
          (2, 3, 1, 130, 33, 17), (1, 2, 1, 150, 100, 200), (1, 2, 2, 17, 1, 1), (1, 2, 2, 129, 200, 5), (1, 4, 2, 70, 96, 512)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype,gate", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("state,last", [(False, False), (True, True)])
def test_gradients(gpu_case, shape, dtype, gate, state, last):
    check_all(*inputs(shape, dtype, gate, sum(shape), state, last))


# many blocks of columns: the scans' form of one wave a block
@pytest.mark.parametrize("shape", [(32, 8, 8, 70, 64, 64), (16, 8, 4, 130, 128, 100), (32, 8, 8, 65, 256, 40)])
@pytest.mark.parametrize("dtype,gate", [(BF16, BF16), (F16, F16), (F32, F32)])
def test_gradients_of_many_heads(gpu_case, shape, dtype, gate):
    check_all(*inputs(shape, dtype, gate, sum(shape), True, True))


def test_last_state_alone(gpu_case):
    x, _, dc = inputs((1, 2, 2, 100, 64, 32), F32, F32, 3)
    check_all(x, None, dc)


def test_strong_decay_and_resets(gpu_case):
    """Resets cut the gradients; padding tokens (g and beta 0) get dbeta of their own and pass the others' on."""
    x, dh, dc = inputs((1, 2, 2, 150, 64, 48), F32, F32, 7, strong=True)
    x[3][:, :, 70:100] = 0
    x[4][:, :, 70:100] = 0
    for t in (0, 40, 64, 127, 128):
        x[3][:, :, t] = -60.0  # exp(-60) = 9e-27: finite, so that the 64-bit gradient of g has no inf * 0
    check_all(x, dh, dc)
    import xlstm_hip
    y = [t.clone() for t in x]
    for t in (0, 40, 64, 127, 128):
        y[3][:, :, t] = -torch.inf
    got = gradients(lambda *z: xlstm_hip.gated_delta_chunkwise(*z, return_last_states=True), y, dh, dc)
    assert all(bool(torch.isfinite(t).all()) for t in got)
    assert float(got[5].abs().max()) == 0  # the initial state is behind a reset


@pytest.mark.parametrize("ks,vs,cs,ds", [(1e-3, 1.0, 1.0, 1.0), (1.0, 1e6, 1e6, 1e-6), (1.0, 1e-6, 1e-6, 1e6), (1.0, 1e8, 1e8, 1e8)])
def test_ranges(gpu_case, ks, vs, cs, ds):
    (q, k, v, g, beta, c0), dh, dc = inputs((1, 2, 2, 140, 64, 48), F32, F32, 5)
    check_all((q, k * ks, v * vs, g, beta, c0 * cs), dh * ds, dc * ds)


def test_columns_of_far_sizes(gpu_case):
    """Blocks of 16 columns with scales of their own meet in one sum."""
    (q, k, v, g, beta, c0), dh, dc = inputs((1, 1, 1, 100, 64, 64), F32, F32, 6)
    size = torch.cat([torch.full((16,), s) for s in (1e4, 1.0, 1e-4, 1e2)]).to(dev())
    check_all((q, k, v * size, g, beta, c0 * size), dh / size, dc / size)


def test_zeros(gpu_case):
    x, dh, dc = inputs((1, 2, 2, 70, 64, 32), F32, F32, 9)
    import xlstm_hip
    fn = lambda *y: xlstm_hip.gated_delta_chunkwise(*y, return_last_states=True)  # noqa: E731
    got = gradients(fn, x, torch.zeros_like(dh), torch.zeros_like(dc))
    assert all(float(t.abs().max()) == 0 for t in got)
    for i in range(3):
        y = list(x)
        y[i] = torch.zeros_like(y[i])
        check_all(y, dh, dc)


def test_differences(gpu_case):
    """The gradient along a direction against the loss's central difference: losses in float64 of float32 outputs of 40 tokens, a
    step of 1e-2.  The difference's own error is step^2 / 6 of a third derivative of the loss's size (1e-4 / 6 x a few), and the
    outputs' float32 errors over the step (5e-6 / 1e-2): 2e-3 of the loss's size."""
    import xlstm_hip
    x, dh, dc = inputs((1, 2, 1, 40, 32, 16), F32, F32, 4)
    fn = lambda *y: xlstm_hip.gated_delta_chunkwise(*y, return_last_states=True)  # noqa: E731
    got = gradients(fn, x, dh, dc)

    def loss(y):
        h, c = fn(*y)
        return float((h.double() * dh.double()).sum() + (c.double() * dc.double()).sum())

    size = float(dh.norm() + dc.norm())
    for i in range(6):
        r = torch.randn(x[i].shape, generator=torch.Generator().manual_seed(i)).to(dev())
        r = r / r.norm()
        up, down = (loss([t + s * 1e-2 * r if j == i else t for j, t in enumerate(x)]) for s in (1, -1))
        slope = (up - down) / 2e-2
        assert abs(slope - float((got[i].double() * r.double()).sum())) <= 2e-3 * size, NAMES[i]


def test_expanded_and_strided_inputs(gpu_case):
    import xlstm_hip
    x, dh, dc = inputs((2, 4, 4, 90, 64, 48), F32, F32, 8)
    fn = lambda *y: xlstm_hip.gated_delta_chunkwise(*y, return_last_states=True)  # noqa: E731
    want = gradients(fn, x, dh, dc)
    y = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in x[:5]] + [x[5]]
    for a, b in zip(gradients(fn, y, dh.transpose(2, 3).contiguous().transpose(2, 3), dc), want):
        assert torch.equal(a, b)
    q1 = x[0][:, :1].clone().requires_grad_(True)  # one query head for all
    h, c = fn(q1.expand_as(x[0]), *x[1:])
    (got,) = torch.autograd.grad((h, c), (q1,), (dh, dc))
    full = gradients(fn, (q1.detach().expand_as(x[0]).contiguous(), *x[1:]), dh, dc)[0]
    assert torch.equal(got, full.sum(1, keepdim=True))
    # a gradient of sum() is expanded from one value
    z = [t.clone().requires_grad_(True) for t in x[:5]]
    xlstm_hip.gated_delta_chunkwise(*z, x[5]).sum().backward()
    a = gradients(lambda *w: (xlstm_hip.gated_delta_chunkwise(*w, x[5]), None), z, torch.ones_like(dh), None)
    assert all(torch.equal(t.grad, u) for t, u in zip(z, a))


def test_some_gradients(gpu_case):
    """Inputs that want none; the same tensor as query and key; no gradient of the state asked for."""
    import xlstm_hip
    x, dh, dc = inputs((1, 2, 2, 70, 64, 32), F32, F32, 10)
    fn = lambda *y: xlstm_hip.gated_delta_chunkwise(*y, return_last_states=True)  # noqa: E731
    want = gradients(fn, x, dh, dc)
    v = x[2].clone().requires_grad_(True)
    h, c = fn(x[0], x[1], v, *x[3:])
    (dv,) = torch.autograd.grad((h, c), (v,), (dh, dc))
    assert torch.equal(dv, want[2])
    k = x[1].clone().requires_grad_(True)
    h, c = fn(k, k, *x[2:])
    (dk,) = torch.autograd.grad((h, c), (k,), (dh, dc))
    both = gradients(fn, (x[1], x[1], *x[2:]), dh, dc)
    assert torch.equal(dk, both[0] + both[1])


def test_deterministic_and_other_stream(gpu_case):
    import xlstm_hip
    x, dh, dc = inputs((2, 4, 2, 300, 64, 64), BF16, BF16, 11)
    fn = lambda *y: xlstm_hip.gated_delta_chunkwise(*y, return_last_states=True)  # noqa: E731
    want = gradients(fn, x, dh, dc)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            got.append(gradients(fn, x, dh, dc))
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, want))


def test_no_tokens(gpu_case):
    import xlstm_hip
    x, dh, dc = inputs((1, 2, 2, 3, 64, 32), F32, F32, 12)
    y = [t[:, :, :0] for t in x[:5]] + [x[5]]
    got = gradients(lambda *z: xlstm_hip.gated_delta_chunkwise(*z, return_last_states=True), y, dh[:, :, :0], dc)
    assert torch.equal(got[5], dc) and got[0].numel() == 0


def test_long(gpu_case):
    """2000 tokens, shared heads, against the 64-bit recurrence."""
    check_all(*inputs((1, 4, 2, 2000, 64, 32), F32, F32, 13))


@pytest.mark.parametrize("shape", [(1, 2, 2, 500, 64, 64), (2, 2, 1, 130, 128, 100), (1, 1, 1, 200, 256, 32)])
def test_float16_is_off_by_its_rounding(gpu_case, shape):
    """float16's operands in the backward are pairs (2^-22): by the bar's count 10 x (2^-22 + 4.5 2^-24) = 5.1e-6 of the parts' norm
    beside the gradient's own rounding to float16 (2e-4 in norm), of which 2 parts' and the cancellation of dg's sums (20 for keys of
    norm 1 and decays near 1) make 2e-4 at most.  One plane's 10 x 2^-11 would be 10 to 20 times that."""
    B, NH, NHK, S, DK, DV = shape
    import xlstm_hip
    r = torch.Generator().manual_seed(S)
    n = lambda *s: torch.randn(*s, generator=r)  # noqa: E731
    unit = lambda t: torch.nn.functional.normalize(t, dim=-1)  # noqa: E731
    x = [t.to(F16).to(dev()) for t in (unit(n(B, NHK, S, DK)), unit(n(B, NHK, S, DK)), n(B, NH, S, DV), -0.2 * torch.rand(B, NH, S, generator=r),
                                       torch.rand(B, NH, S, generator=r))] + [None]
    dh = n(B, NH, S, DV).to(F16).to(dev())
    scale = DK ** -0.5
    got = gradients(lambda q, k, v, g, b, c: xlstm_hip.gated_delta_chunkwise(q, k, v, g, b, c, scale, True), x, dh, None)
    want = gradients(lambda q, k, v, g, b, c: plain(q, k, v, g, b, c, scale), x, dh, None, torch.float64)
    for name, a, w in zip(NAMES, got, want):
        err, rounding = float((a.double() - w).norm()), float((w.to(F16).double() - w).norm())
        assert err <= rounding + 2e-4 * float(w.norm()), f"{name}: {err / float(w.norm()):.2e}"
