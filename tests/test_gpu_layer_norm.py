"""Layer norm and its gradients on the GPU, against the formula in 64 bits and against differences.

Bars, from the arithmetic (u = 2^-24): a float32 sum of n terms in any order is off by at most n u times the sum of
their magnitudes; per-row sums here run D / 64 + 24 terms deep at most (a lane's own values, then a tree), so with
k = (D / 64 + 24) u the mean is off by k mean|x| and h = (x - mean) rstd by e_h = k (2 |h| + 2 max|x| rstd); a sum over
N tokens by (N + 16) u.  Each output then has one rounding of its type (half a unit in its last place)."""

import pytest
import torch

from helpers import dev, half_ulp

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def reference(x, w, b, dy, eps):
    """x [tokens, H, D], w / b [H, D] or None: (value, bar) of y, dx, dw, db; dy None: of y alone."""
    x = x.double()
    D = x.shape[-1]
    w1 = torch.ones(x.shape[1:], dtype=torch.float64, device=x.device) if w is None else w.double()
    b1 = torch.zeros_like(w1) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    h = (x - mean) * rstd
    y = h * w1 + b1
    k = (D / 64 + 24) * U
    e_h = k * (2 * h.abs() + 2 * x.abs().amax(-1, keepdim=True) * rstd)
    out = [(y, e_h * w1.abs() + 2 * U * ((h * w1).abs() + b1.abs()))]
    if dy is None:
        return out
    dy = dy.double()
    g = dy * w1
    c1, c2 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    dx = rstd * (g - c1 - h * c2)
    m1, m2 = g.abs().mean(-1, keepdim=True), (g * h).abs().mean(-1, keepdim=True)
    out.append((dx, rstd * (4 * k * (g.abs() + m1 + h.abs() * m2) + e_h * m2 + h.abs() * (g.abs() * e_h).mean(-1, keepdim=True))))
    n = (x.shape[0] + 16) * U
    out.append(((dy * h).sum(0), n * (dy * h).abs().sum(0) + (dy.abs() * e_h).sum(0)))
    out.append((dy.sum(0), n * dy.abs().sum(0)))
    return out


def check(got, want, bar, what):
    err = (got.detach().double() - want).abs() - bar - half_ulp(want, got.dtype).to(want.device)
    assert got.shape == want.shape and bool((err <= 0).all()), f"{what}: {float(err.max()):.3e} over the bar"


def inputs(tokens, H, D, dtype, param, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(tokens, H, D, generator=g) * 1.5 + torch.randn(D, generator=g)).to(dtype).to(dev())
    w = (1 + 0.2 * torch.randn(H, D, generator=g)).to(param).to(dev())
    b = (0.3 * torch.randn(H, D, generator=g)).to(param).to(dev())
    dy = torch.randn(tokens, H, D, generator=g).to(dtype).to(dev())
    return x, w, b, dy


# one value, less than a vector, one vector, odd, every team size and register count, past the registers
WIDTHS = [1, 5, 8, 64, 100, 129, 512, 777, 1024, 1333, 2048, 4096, 5503, 8192, 10944, 16392, 33000, 70001]


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype,param", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F32, F32)])
def test_forward_and_gradients(gpu_case, D, dtype, param):
    import xlstm_hip
    tokens = 3 if D > 20000 else 37
    x, w, b, dy = (t.squeeze(1) if t.dim() == 3 else t[0] for t in inputs(tokens, 1, D, dtype, param, D))
    for t in (x, w, b):
        t.requires_grad_(True)
    y = xlstm_hip.layer_norm(x, w, b, 1e-5)
    got = (y, *torch.autograd.grad(y, (x, w, b), dy))
    want = reference(x.detach()[:, None], w.detach()[None], b.detach()[None], dy[:, None], 1e-5)
    assert got[2].dtype == got[3].dtype == param and got[1].dtype == y.dtype == dtype
    for a, (v, bar), name in zip(got, want, ("y", "dx", "dw", "db")):
        v, bar = (t.squeeze(0 if name in ("dw", "db") else 1) for t in (v, bar))
        check(a, v, bar, name)


# one token, few, more than the slices of the weight's gradient, many
@pytest.mark.parametrize("tokens", [1, 2, 5, 255, 513, 4097, 20000])
@pytest.mark.parametrize("D,dtype", [(96, F32), (520, BF16), (1333, F16)])
def test_token_counts(gpu_case, tokens, D, dtype):
    import xlstm_hip
    x, w, b, dy = (t.squeeze(1) if t.dim() == 3 else t[0] for t in inputs(tokens, 1, D, dtype, F32, tokens))
    for t in (x, w, b):
        t.requires_grad_(True)
    y = xlstm_hip.layer_norm(x, w, b, 1e-6)
    got = (y, *torch.autograd.grad(y, (x, w, b), dy))
    want = reference(x.detach()[:, None], w.detach()[None], b.detach()[None], dy[:, None], 1e-6)
    for a, (v, bar), name in zip(got, want, ("y", "dx", "dw", "db")):
        check(a, *(t.squeeze(0 if name in ("dw", "db") else 1) for t in (v, bar)), name)


@pytest.mark.parametrize("B,NH,S,DH", [(1, 1, 1, 64), (2, 4, 33, 128), (3, 8, 17, 512), (2, 3, 50, 65), (1, 2, 300, 1100)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads_first", [True, False])
def test_heads(gpu_case, B, NH, S, DH, dtype, heads_first):
    import xlstm_hip
    x, w, b, dy = inputs(B * S, NH, DH, dtype, dtype, DH + S)
    h = x.view(B, S, NH, DH)
    if heads_first:
        h = h.transpose(1, 2).contiguous()
    h, w1, b1 = (t.detach().requires_grad_(True) for t in (h, w.reshape(-1), b.reshape(-1)))
    y = xlstm_hip.multi_head_layer_norm(h, w1, b1, 1e-6, heads_first)
    dh, dw, db = torch.autograd.grad(y, (h, w1, b1), dy.view(B, S, NH * DH))
    assert dh.stride() == h.stride() and y.is_contiguous()
    got = (y.view(B * S, NH, DH), (dh.transpose(1, 2) if heads_first else dh).reshape(B * S, NH, DH), dw.view(NH, DH),
           db.view(NH, DH))
    for a, (v, bar), name in zip(got, reference(x, w, b, dy, 1e-6), ("y", "dh", "dw", "db")):
        check(a, v, bar, name)


def _strided(kind, dtype):
    """x of other strides than a fresh tensor's, [..., 200]."""
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(dev())  # noqa: E731
    return {"columns": lambda: r(9, 700)[:, 33:233], "odd start": lambda: r(9 * 200 + 1)[1:].view(9, 200),
            "every third row": lambda: r(27, 200)[::3], "two axes swapped": lambda: r(4, 6, 200).transpose(0, 1),
            "three axes": lambda: r(3, 4, 5, 200).permute(2, 0, 1, 3), "broadcast rows": lambda: r(1, 200).expand(6, 200),
            "broadcast values": lambda: r(6, 1).expand(6, 200), "values apart": lambda: r(200, 9).t(),
            "one row": lambda: r(200)}[kind]()


@pytest.mark.parametrize("kind", ["columns", "odd start", "every third row", "two axes swapped", "three axes", "broadcast rows",
                                  "broadcast values", "values apart", "one row"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides(gpu_case, kind, dtype):
    import xlstm_hip
    x = _strided(kind, dtype).requires_grad_(True)
    _, w, b, _ = inputs(1, 1, 200, dtype, dtype, 3)
    dy = torch.randn(x.shape[-1], *x.shape[:-1], generator=torch.Generator().manual_seed(1)).to(dtype).to(dev()).movedim(0, -1)
    y = xlstm_hip.layer_norm(x, w[0], b[0])
    (dx,) = torch.autograd.grad(y, x, dy)
    want = reference(x.detach().reshape(-1, 1, 200), w, b, dy.reshape(-1, 1, 200), 1e-5)
    check(y.reshape(-1, 1, 200), *want[0], "y")
    check(dx.reshape(-1, 1, 200), *want[1], "dx")


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("wanted", ["x", "w", "b", "xw"])
def test_optional_arguments_and_gradients(gpu_case, weight, bias, wanted):
    import xlstm_hip
    x, w, b, dy = inputs(21, 1, 300, BF16, F32, 5)
    x1, w1, b1 = x[:, 0].clone(), w[0].clone() if weight else None, b[0].clone() if bias else None
    given = {"x": x1, "w": w1, "b": b1}
    asked = [c for c in wanted if given[c] is not None]
    if not asked:
        pytest.skip("the argument that the gradient is asked of is left out")
    for c in asked:
        given[c].requires_grad_(True)
    y = xlstm_hip.layer_norm(x1, w1, b1)
    got = torch.autograd.grad(y, [given[c] for c in asked], dy[:, 0])
    want = reference(x, w if weight else None, b if bias else None, dy, 1e-5)
    check(y[:, None], *want[0], "y")
    for a, c in zip(got, asked):
        v, bar = want[1 + "xwb".index(c)]
        check(a[:, None] if c == "x" else a[None], v, bar, "d" + c)


def test_gradient_against_differences(gpu_case):
    """The directional derivative of sum(y c) from central differences of the kernel's own float32 outputs: off by the
    outputs' bars over the step, and by what the step itself leaves out (taken from the formula in 64 bits)."""
    import xlstm_hip
    x, w, b, c = inputs(4, 1, 64, F32, F32, 11)
    g = torch.Generator().manual_seed(12)
    v = [torch.randn(t.shape, generator=g).to(dev()) for t in (x, w, b)]
    step = 2.0 ** -6
    leaves = [t.clone().requires_grad_(True) for t in (x[:, 0], w[0], b[0])]
    grads = torch.autograd.grad(xlstm_hip.layer_norm(*leaves), leaves, c[:, 0])
    slope = sum(float((a.double() * d.double().view(a.shape)).sum()) for a, d in zip(grads, v))
    ends, ends64, slack = [], [], 0.0
    for s in (step, -step):
        moved = [t + s * d for t, d in zip((x, w, b), v)]
        y = xlstm_hip.layer_norm(moved[0][:, 0], moved[1][0], moved[2][0])
        ends.append(float((y.double() * c[:, 0].double()).sum()))
        exact, bar = reference(*moved, None, 1e-5)[0]
        ends64.append(float((exact * c.double()).sum()))
        slack += float((bar * c.abs().double()).sum()) / (2 * step)
    want = reference(x, w, b, c, 1e-5)
    slope64 = sum(float((want[1 + i][0].reshape(v[i].shape) * v[i].double()).sum()) for i in range(3))
    slack += sum(float((want[1 + i][1].reshape(v[i].shape) * v[i].abs().double()).sum()) for i in range(3))
    # the steps are rounded to float32 when they are added: a unit in the last place of each moved value
    slack += sum(float((want[1 + i][0].reshape(v[i].shape).abs() * 4 * U * t.abs().double()).sum()) / step
                 for i, t in enumerate((x, w, b)))
    left_out = abs((ends64[0] - ends64[1]) / (2 * step) - slope64)
    assert abs((ends[0] - ends[1]) / (2 * step) - slope) <= 1.01 * left_out + 2 * slack
    assert left_out + slack < 0.2 * abs(slope)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_tokens(gpu_case, dtype):
    import xlstm_hip
    x, w, b = torch.empty(0, 64, dtype=dtype, device=dev()), torch.ones(64, device=dev()), torch.ones(64, device=dev())
    for t in (x, w, b):
        t.requires_grad_(True)
    y = xlstm_hip.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == dx.shape == (0, 64) and not dw.any() and not db.any()


@pytest.mark.parametrize("D", [64, 1333, 33000])
def test_special_values_stay_in_their_row(gpu_case, D):
    """A NaN or an infinity makes its own row NaN and no other; a constant row is its bias; far from zero, the variance
    does not cancel."""
    import xlstm_hip
    x, w, b, _ = inputs(5, 1, D, F32, F32, 2)
    x, w, b = x[:, 0], w[0], b[0]
    x[1, D // 2], x[2, 0], x[3] = float("nan"), float("inf"), 17.0
    x[4] += 1000.0
    y = xlstm_hip.layer_norm(x, w, b)
    assert bool(y[1].isnan().all()) and bool(y[2].isnan().all())
    assert torch.equal(y[3], b)
    want = reference(x[[0, 4], None], w[None], b[None], None, 1e-5)[0]
    check(y[[0, 4], None], *want, "y")


def test_rows_past_32_bits(gpu_case):
    """Rows more than 2^31 values apart, in x and in dx."""
    import xlstm_hip
    apart = 2 ** 31 + 24
    buf = torch.zeros(apart + 128, dtype=BF16, device=dev())
    rows, w, b, dy = inputs(2, 1, 128, BF16, BF16, 4)
    x = buf.as_strided((2, 128), (apart, 1))
    x.copy_(rows[:, 0])
    x.requires_grad_(True)
    y = xlstm_hip.layer_norm(x, w[0], b[0])
    (dx,) = torch.autograd.grad(y, x, dy[:, 0])
    want = reference(rows, w, b, dy, 1e-5)
    check(y[:, None], *want[0], "y")
    check(dx[:, None], *want[1], "dx")


def test_other_stream_and_same_bits(gpu_case):
    """On a stream of its own, behind the work that makes its input there; the same bits every time."""
    import xlstm_hip
    x, w, b, dy = (t.squeeze(1) if t.dim() == 3 else t[0] for t in inputs(5000, 1, 1024, BF16, F32, 6))

    def step():
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = xlstm_hip.layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(first, again))


def test_graph_replays(gpu_case):
    import xlstm_hip
    x, w, b, dy = (t.squeeze(1) if t.dim() == 3 else t[0] for t in inputs(300, 1, 520, BF16, F32, 8))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]

    def step():
        y = xlstm_hip.layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        with torch.no_grad():
            leaves[0].copy_(x * (1 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(held, step())), f"replay {k}"


@pytest.mark.parametrize("layout", [0, 1, 2])
@pytest.mark.parametrize("order", ["as made", "last axis first", "heads first", "three axes", "every other", "broadcast"])
def test_gradient_lies_as_traced(gpu_case, layout, order):
    """dx has the strides that a traced program takes it to have, whatever x's are, and the same bits."""
    import xlstm_hip  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    op = torch.ops.xlstm_hip.layer_norm_bwd.default
    g = torch.Generator().manual_seed(5)
    B, M, N, D = 3, 4, 6, 40
    x = torch.randn(B, M, N, D, generator=g).to(dev())
    x = {"as made": lambda: x, "last axis first": lambda: x.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0),
         "heads first": lambda: x.transpose(1, 2).contiguous().transpose(1, 2),
         "three axes": lambda: x.permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3),
         "every other": lambda: torch.cat([x, x], 2)[:, :, ::2], "broadcast": lambda: x[:, :1].expand(B, M, N, D)}[order]()
    heads = (1, M, N)[layout]
    shape = (x.shape, (B, N, M * D), (B, M, N * D))[layout]
    dy = torch.randn(shape, generator=g).to(dev())
    w = torch.randn(heads * D, generator=g).to(dev())
    stats = torch.ops.xlstm_hip.layer_norm.default(x, w, None, 1e-5, layout)[1]
    dx = op(dy, x, stats, w, None, layout, [True, True, False])[0]
    with FakeTensorMode() as mode:
        traced = op(*(mode.from_tensor(t) for t in (dy, x, stats, w)), None, layout, [True, True, False])[0]
    assert dx.shape == traced.shape and dx.stride() == traced.stride()
    plain = op(dy, x.contiguous(), stats, w, None, layout, [True, True, False])[0]
    assert torch.equal(dx, plain)


def test_modules_train_on_it(gpu_case):
    """MultiHeadLayerNorm, whose kernel without a gradient has none, differentiates through this norm; without a
    gradient it gives what it gave."""
    import xlstm_hip
    x, w, b, dy = inputs(2 * 30, 4, 96, BF16, BF16, 9)
    norm = xlstm_hip.MultiHeadLayerNorm(4, 96, use_bias=True).to(dev()).to(BF16)
    with torch.no_grad():
        norm.weight.copy_(w.reshape(-1))
        norm.bias.copy_(b.reshape(-1))
        plain = norm(x.view(2, 30, 4, 96))
        assert torch.equal(plain, xlstm_hip.group_norm(x.view(60, -1), 4, norm.weight, norm.bias, 1e-6).view(2, 30, -1))
    y = norm(x.view(2, 30, 4, 96))
    dw, db = torch.autograd.grad(y, (norm.weight, norm.bias), dy.view(2, 30, -1))
    want = reference(x, w, b, dy, 1e-6)
    for a, (v, bar), name in zip((y.view(60, 4, 96), dw.view(4, 96), db.view(4, 96)), (want[0], want[2], want[3]),
                                 ("y", "dw", "db")):
        check(a, v, bar, name)


@pytest.mark.parametrize("what", ["weight shape", "bias shape", "dtypes", "weight dtype", "heads", "double backward"])
def test_refusals(gpu_case, what):
    import xlstm_hip
    x, w = torch.randn(4, 64, device=dev(), dtype=BF16), torch.ones(64, device=dev())
    if what == "weight shape":
        with pytest.raises(ValueError, match="weight"):
            xlstm_hip.layer_norm(x, w[:32])
    elif what == "bias shape":
        with pytest.raises(ValueError, match="bias"):
            xlstm_hip.layer_norm(x, w, torch.ones(2, 64, device=dev()))
    elif what == "dtypes":
        with pytest.raises(ValueError, match="share"):
            xlstm_hip.layer_norm(x, w, w.to(BF16))
    elif what == "weight dtype":
        with pytest.raises(ValueError, match="dtype"):
            xlstm_hip.layer_norm(x, w.to(F16))
        with pytest.raises(ValueError, match="dtype"):
            xlstm_hip.layer_norm(x.double(), None)
    elif what == "heads":
        with pytest.raises(ValueError, match="weight"):
            xlstm_hip.multi_head_layer_norm(x.view(1, 2, 2, 64), w)
        with pytest.raises(ValueError, match="4-D"):
            xlstm_hip.multi_head_layer_norm(x, w)
    else:
        x.requires_grad_(True)
        (dx,) = torch.autograd.grad(xlstm_hip.layer_norm(x).float().sum(), x, create_graph=True)
        if dx.requires_grad:
            with pytest.raises(RuntimeError):
                torch.autograd.grad(dx.float().square().sum(), x)
