"""The gated linear unit's GELU where its gate is far below zero: a (1 + erf(a / sqrt 2)) / 2 cancels there, and the result is still right to
its own bits.

Bar: the products are exact (one term each, the other factor 1), erfc is off by 8 units of 2^-24 relative, its argument by 2 (the constant
and the product), which it multiplies by a^2; then the result's own rounding."""

import pytest
import torch

from helpers import dev, half_ulp

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
U = 2.0 ** -24


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("dtype,lowest", [(BF16, -9.0), (F16, -4.0)])
def test_gelu_far_below_zero(gpu_case, T, dtype, lowest):
    import xlstm_hip
    a = torch.linspace(lowest, 1.0, 200).to(dtype).to(dev())
    x = torch.zeros(T, 8, dtype=dtype, device=dev())
    x[0, 0] = 1
    wg, wu = (torch.zeros(200, 8, dtype=dtype, device=dev()) for _ in range(2))
    wg[:, 0], wu[:, 0] = a, 1
    want = a.double() * torch.special.erfc(-a.double() * 0.5 ** 0.5) / 2
    bar = (8 + 2 * a.double() ** 2) * U * want.abs()
    ulp = half_ulp(want, dtype).clamp_min(2.0 ** -25 if dtype == F16 else 0.0).to(dev())
    h = xlstm_hip.gated_linear_unit(x, wg, wu, "gelu")
    assert bool(((h[0].double() - want).abs() <= bar + ulp).all()), "h"
    w = [t.clone().requires_grad_(True) for t in (wg, wu)]
    (dwu,) = torch.autograd.grad(xlstm_hip.gated_linear_unit(x, *w, "gelu")[0].sum(), w[1:])  # act(a), rounded once as du and not again
    assert bool(((dwu[:, 0].double() - want).abs() <= bar + ulp).all()), "dwu"
