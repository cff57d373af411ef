"""The gated linear unit on the GPU against the formula in 64 bits, and its gradients, also against differences.

Bars, with u = 2^-24 and r = eps / 2 of the type (bf16 2^-9 of a value's binade at most, taken as half an ulp): a product's sum
of n float32 terms is off by n u times the sum of their magnitudes at most; act by 8 u relative (exp2, the reciprocal, erf) and 1.1
times its argument's error (its largest slope).  da and du are rounded to the type (eps / 2 relative), as are the results."""

import pytest
import torch

from helpers import dev, half_ulp

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
U = 2.0 ** -24


def act(a, kind):
    return torch.nn.functional.silu(a) if kind == "silu" else torch.nn.functional.gelu(a)


def inputs(T, D, F, dtype, seed, scale=1.0):
    r = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=r)  # noqa: E731
    return [t.to(dtype).to(dev()) for t in (n(T, D) * scale, n(F, D) * D ** -0.5, n(F, D) * D ** -0.5, n(T, F))]


def reference(x, wg, wu, dh, kind):
    """(value, bar without its own rounding) of h, dx, dwg, dwu."""
    eps = torch.finfo(x.dtype).eps / 2
    x, wg, wu, dh = (t.double() for t in (x, wg, wu, dh))
    D = x.shape[1]
    a, u = (x @ w.t() for w in (wg, wu))
    ea, eu = (D * U * (x.abs() @ w.abs().t()) for w in (wg, wu))
    a.requires_grad_(True)
    f = act(a, kind)
    (slope,) = torch.autograd.grad(f.sum(), a)
    a, f = a.detach(), f.detach()
    ef = 1.1 * ea + 8 * U * f.abs()
    out = [(f * u, ef * u.abs() + f.abs() * eu + ef * eu)]
    da, du = dh * u * slope, dh * f
    # act' is off by 0.8 ea at most (its own largest slope) and 8 u
    eda = dh.abs() * (eu * slope.abs() + u.abs() * (0.8 * ea + 8 * U)) + da.abs() * eps
    edu = dh.abs() * ef + du.abs() * eps
    if x.dtype == F16 or eps == torch.finfo(F16).eps / 2:  # f16 numbers below 2^-14 are 2^-24 apart
        eda, edu = eda + 2.0 ** -25, edu + 2.0 ** -25
    n = 2 * wg.shape[0] * U
    out.append((da @ wg + du @ wu, eda @ wg.abs() + edu @ wu.abs() + n * (da.abs() @ wg.abs() + du.abs() @ wu.abs())))
    n = (x.shape[0] + 64) * U
    for d, e in ((da, eda), (du, edu)):
        out.append((d.t() @ x, e.t() @ x.abs() + n * (d.abs().t() @ x.abs())))
    return out


def check(got, want, bar, what):
    ulp = half_ulp(want, got.dtype).clamp_min(2.0 ** -25 if got.dtype == F16 else 0.0).to(want.device)
    err = (got.detach().double() - want).abs() - bar - ulp
    # what lies past the type's largest value and half a step (f16: 65520) rounds to infinity
    most = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    err = torch.where(torch.isinf(got) & (got.sign() == want.sign()) & (want.abs() + bar >= most), torch.zeros_like(err), err)
    assert got.shape == want.shape and bool((err <= 0).all()), f"{what}: {float(err.max()):.3e} over the bar"


def run(x, wg, wu, dh, kind="silu"):
    import xlstm_hip
    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    h = xlstm_hip.gated_linear_unit(*leaves, kind)
    return (h, *torch.autograd.grad(h, leaves, dh))


NAMES = ("h", "dx", "dwg", "dwu")
# one token, the streaming form's rows, tiles' edges, sizes that nothing divides, rows of odd lengths, one value
SIZES = [(1, 64, 64), (1, 1, 1), (3, 8, 5), (16, 512, 100), (17, 72, 33), (64, 64, 64), (65, 128, 129), (100, 1000, 273),
         (130, 33, 257), (257, 200, 300), (300, 264, 520), (513, 7, 70), (1000, 320, 136)]


@pytest.mark.parametrize("T,D,F", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_values_and_gradients(gpu_case, T, D, F, dtype, kind):
    import xlstm_hip
    x, wg, wu, dh = inputs(T, D, F, dtype, T + D + F)
    want = reference(x, wg, wu, dh, kind)
    for g, (v, bar), name in zip(run(x, wg, wu, dh, kind), want, NAMES):
        assert g.dtype == dtype
        check(g, v, bar, name)
    check(xlstm_hip.gated_linear_unit(x, wg, wu, kind), *want[0], "h without a gradient")


@pytest.mark.parametrize("T,D,F", [(2048, 512, 2048), (4096, 256, 1024), (700, 2048, 5504), (128, 1024, 2752), (8192, 64, 96)])
def test_large_tiles(gpu_case, T, D, F):
    """Sizes that take the larger tiles."""
    x, wg, wu, dh = inputs(T, D, F, BF16, T)
    for g, (v, bar), name in zip(run(x, wg, wu, dh), reference(x, wg, wu, dh, "silu"), NAMES):
        check(g, v, bar, name)


@pytest.mark.parametrize("T,D,F", [(70, 136, 2731), (5, 264, 5504), (777, 512, 5504), (4200, 72, 130), (2500, 200, 1025), (4096, 512, 256)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_sums_in_parts(gpu_case, T, D, F, dtype):
    """Few tiles and a long sum: dx over the features, the weights' over the tokens, in parts that do not divide their slices."""
    x, wg, wu, dh = inputs(T, D, F, dtype, T + 1)
    first = run(x, wg, wu, dh)
    for g, (v, bar), name in zip(first, reference(x, wg, wu, dh, "silu"), NAMES):
        check(g, v, bar, name)
    assert all(torch.equal(a, b) for a, b in zip(first, run(x, wg, wu, dh)))


@pytest.mark.parametrize("M", [1, 2, 7, 8, 15, 16])
@pytest.mark.parametrize("D,F", [(4096, 1000), (24, 17), (2048, 5504)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_few_tokens(gpu_case, M, D, F, dtype):
    import xlstm_hip
    x, wg, wu, dh = inputs(M, D, F, dtype, M + D)
    check(xlstm_hip.gated_linear_unit(x, wg, wu), *reference(x, wg, wu, dh, "silu")[0], "h")


@pytest.mark.parametrize("T", [5, 70])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_wide_range(gpu_case, T, dtype):
    """Gates far out on both sides: silu's exp overflows and underflows."""
    import xlstm_hip
    x, wg, wu, dh = inputs(T, 64, 96, dtype, 1, scale=100.0)
    h = xlstm_hip.gated_linear_unit(x, wg, wu)
    want = reference(x, wg, wu, dh, "silu")
    assert not bool(torch.isnan(h).any())  # products past 65504 are infinite in float16
    for g, (v, bar), name in zip(run(x, wg, wu, dh), want, NAMES):
        check(g, v, bar, name)


def test_not_finite_stays_in_its_rows(gpu_case):
    """NaN and infinity in one token or one weight's row, also at the ends of padded tiles and slices."""
    import xlstm_hip
    for T, D in ((70, 104), (9, 104), (70, 33)):
        x, wg, wu, _ = inputs(T, D, 80, BF16, 2)
        want = xlstm_hip.gated_linear_unit(x, wg, wu)
        for value in (float("nan"), float("inf")):
            y = x.clone()
            y[3, D - 1] = value
            h = xlstm_hip.gated_linear_unit(y, wg, wu)
            keep = torch.arange(T, device=dev()) != 3
            assert torch.equal(h[keep], want[keep]) and not bool(torch.isfinite(h[3]).any())
            w = wu.clone()
            w[79, 0] = value
            h = xlstm_hip.gated_linear_unit(x, wg, w)
            assert torch.equal(h[:, :79], want[:, :79]) and not bool(torch.isfinite(h[:, 79]).any())


def test_shapes_and_strides(gpu_case):
    import xlstm_hip
    x, wg, wu, _ = inputs(30, 64, 40, BF16, 3)
    want = xlstm_hip.gated_linear_unit(x, wg, wu)
    assert torch.equal(xlstm_hip.gated_linear_unit(x.view(2, 3, 5, 64), wg, wu), want.view(2, 3, 5, 40))
    assert torch.equal(xlstm_hip.gated_linear_unit(x[0], wg, wu), want[0])
    held = torch.empty(30 * 64 + 1, dtype=BF16, device=dev())
    held[1:] = x.reshape(-1)
    assert torch.equal(xlstm_hip.gated_linear_unit(held[1:].view(30, 64), wg, wu), want)
    assert torch.equal(xlstm_hip.gated_linear_unit(x.t().contiguous().t(), wg.t().contiguous().t(), wu), want)
    both = torch.cat([wg, wu])  # one tensor of both weights
    assert torch.equal(xlstm_hip.gated_linear_unit(x, both[:40], both[40:]), want)
    assert xlstm_hip.gated_linear_unit(x[:0], wg, wu).shape == (0, 40)


def test_no_tokens_gradients(gpu_case):
    x, wg, wu, dh = inputs(4, 64, 40, BF16, 3)
    h, dx, dwg, dwu = run(x[:0], wg, wu, dh[:0])
    assert dx.shape == (0, 64) and float(dwg.abs().max()) == float(dwu.abs().max()) == 0


def test_some_gradients(gpu_case):
    """Any one of the three; one tensor as both weights; a gradient expanded from one value."""
    import xlstm_hip
    x, wg, wu, dh = inputs(70, 64, 40, BF16, 4)
    want = run(x, wg, wu, dh)
    for i in range(3):
        y = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, wg, wu))]
        (g,) = torch.autograd.grad(xlstm_hip.gated_linear_unit(*y), (y[i],), dh)
        assert torch.equal(g, want[1 + i])
    w = wg.detach().requires_grad_(True)
    (g,) = torch.autograd.grad(xlstm_hip.gated_linear_unit(x, w, w), (w,), dh)
    both = run(x, wg, wg, dh)
    assert torch.equal(g, both[2] + both[3])
    y = [t.detach().requires_grad_(True) for t in (x, wg, wu)]
    xlstm_hip.gated_linear_unit(*y).sum().backward()
    assert all(torch.equal(t.grad, g) for t, g in zip(y, run(x, wg, wu, torch.ones_like(dh))[1:]))


def test_differences(gpu_case):
    """Against central differences of the loss over steps of one part in 16 along a direction.  h is rounded to f16, 2^-11 of each of
    T F values of about 1 with random signs: 2^-11 sqrt(T F) / 2 a loss; the difference of two over 1/8 leaves 8 2^-11 |dh|."""
    import xlstm_hip
    x, wg, wu, dh = inputs(40, 64, 48, F16, 5)
    got = run(x, wg, wu, dh)
    loss = lambda *t: float((xlstm_hip.gated_linear_unit(*t).double() * dh.double()).sum())  # noqa: E731
    size = float(dh.double().norm())
    for i, t in enumerate((x, wg, wu)):
        # a direction that f16 holds: a sixteenth of t itself, so t (1 +- 1/16) is off by a rounding of 2^-11 / (1/16) at most
        up, down = (loss(*[(s.double() * (1 + sign / 16)).to(F16) if j == i else s for j, s in enumerate((x, wg, wu))]) for sign in (1, -1))
        slope = float((got[1 + i].double() * t.double()).sum())
        # third derivatives: the slope's own size times (1/16)^2
        assert abs((up - down) * 8 - slope) <= 16 * 2.0 ** -11 * size * 8 + abs(slope) / 256 + size / 256, NAMES[1 + i]


def test_deterministic_and_other_stream(gpu_case):
    x, wg, wu, dh = inputs(300, 520, 264, BF16, 6)
    want = run(x, wg, wu, dh)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            got.append(run(x, wg, wu, dh))
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, want))


def test_nothing_past_the_ends(gpu_case):
    """Results of odd sizes leave what lies behind them alone."""
    import xlstm_hip
    from xlstm_hip import _lib
    lib = _lib.load()
    T, D, F = 67, 72, 43
    x, wg, wu, dh = inputs(T, D, F, BF16, 7)
    want = run(x, wg, wu, dh)
    h = torch.full((T * F + 64,), 7.0, dtype=BF16, device=dev())
    st = torch.cuda.current_stream().cuda_stream
    assert lib.xl_gated_linear_fwd(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), h.data_ptr(), None, None, 0, T, D, F, 0, 1, None, 0, st) == 0
    assert torch.equal(h[:T * F].view(T, F), xlstm_hip.gated_linear_unit(x, wg, wu)) and bool((h[T * F:] == 7).all())
    kept = torch.zeros(2, T, 48, device=dev())
    ws = torch.empty(lib.xl_gated_linear_workspace_size(T, D, F, 1, 1), dtype=torch.uint8, device=dev())
    assert lib.xl_gated_linear_fwd(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), h.data_ptr(), kept[0].data_ptr(), kept[1].data_ptr(), 48, T, D,
                                   F, 0, 1, None, 0, st) == 0
    dx, dg, du = (torch.full((n + 64,), 7.0, dtype=BF16, device=dev()) for n in (T * D, F * D, F * D))
    assert lib.xl_gated_linear_bwd(dh.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), kept[0].data_ptr(), kept[1].data_ptr(), 48,
                                   dx.data_ptr(), dg.data_ptr(), du.data_ptr(), T, D, F, 0, 1, ws.data_ptr(), ws.numel(), st) == 0
    for t, g in zip((dx, dg, du), want[1:]):
        assert torch.equal(t[:g.numel()], g.reshape(-1)) and bool((t[g.numel():] == 7).all())
