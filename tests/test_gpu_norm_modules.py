"""MultiHeadLayerNorm in training and in evaluation: one result, the GroupNorm kernel's, weights of x's type or float32.

Bars as in test_gpu_layer_norm.py."""

import pytest
import torch

from helpers import dev
from test_gpu_layer_norm import BF16, F16, F32, check, inputs, reference

pytestmark = pytest.mark.gpu


def module(NH, DH, w, b):
    import xlstm_hip
    norm = xlstm_hip.MultiHeadLayerNorm(NH, DH, use_bias=True).to(dev()).to(w.dtype)
    with torch.no_grad():
        norm.weight.copy_(w.reshape(-1))
        norm.bias.copy_(b.reshape(-1))
    return norm


@pytest.mark.parametrize("dtype,param", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("B,S,NH,DH", [(2, 30, 4, 96), (1, 1, 2, 64), (3, 7, 4, 512), (2, 9, 3, 65), (1, 5, 2, 6000)])
def test_training_and_evaluation_agree(gpu_case, dtype, param, B, S, NH, DH):
    x, w, b, dy = inputs(B * S, NH, DH, dtype, param, DH)
    norm = module(NH, DH, w, b)
    h = x.view(B, S, NH, DH)
    with torch.no_grad():
        plain = norm(h)
    frozen = [p.detach() for p in (norm.weight, norm.bias)]
    leaf = h.detach().clone().requires_grad_(True)
    y = norm(leaf)
    assert y.shape == (B, S, NH * DH) and y.dtype == dtype and torch.equal(y, plain)
    if param == dtype:
        import xlstm_hip
        assert torch.equal(y, xlstm_hip.group_norm(h.reshape(B * S, -1), NH, *frozen, norm.eps).view_as(y))
    dh, dw, db = torch.autograd.grad(y, (leaf, norm.weight, norm.bias), dy.view(B, S, NH * DH))
    want = reference(x, w, b, dy, norm.eps)
    for a, (v, bar), name in zip((y.view(B * S, NH, DH), dh.view(B * S, NH, DH), dw.view(NH, DH), db.view(NH, DH)), want,
                                 ("y", "dh", "dw", "db")):
        check(a, v, bar, name)


@pytest.mark.parametrize("wanted", ["x", "weight", "frozen"])
@pytest.mark.parametrize("order", ["tokens apart", "heads first"])
def test_module_orders_and_parts(gpu_case, wanted, order):
    """x of other strides, and a gradient of one argument alone."""
    x, w, b, dy = inputs(2 * 12, 4, 40, BF16, BF16, 3)
    norm = module(4, 40, w, b)
    h = x.view(2, 12, 4, 40)
    h = torch.cat([h, h], 3)[..., :40] if order == "tokens apart" else h.transpose(1, 2).contiguous().transpose(1, 2)
    with torch.no_grad():
        plain = norm(h)
    for p in norm.parameters():
        p.requires_grad_(wanted == "weight")
    leaf = h.detach().requires_grad_(wanted == "x")
    y = norm(leaf)
    assert torch.equal(y, plain) and y.requires_grad == (wanted != "frozen")
    want = reference(x, w, b, dy, norm.eps)
    if wanted == "x":
        (dh,) = torch.autograd.grad(y, leaf, dy.view(2, 12, -1))
        check(dh.reshape(24, 4, 40), *want[1], "dh")
    elif wanted == "weight":
        (dw,) = torch.autograd.grad(y, norm.weight, dy.view(2, 12, -1))
        check(dw.view(4, 40), *want[2], "dw")


def test_no_tokens(gpu_case):
    norm = module(4, 40, torch.ones(4, 40, device=dev()), torch.ones(4, 40, device=dev()))
    y = norm(torch.empty(2, 0, 4, 40, device=dev()))
    dw, db = torch.autograd.grad(y, (norm.weight, norm.bias), torch.empty_like(y))
    assert y.shape == (2, 0, 160) and not dw.any() and not db.any()


def test_module_on_the_group_norm_kernel(gpu_case):
    """Without a gradient, against the oracle of the GroupNorm."""
    from helpers import assert_parity
    from oracle import slstm_layers as osl
    x, w, b, _ = inputs(2 * 40, 4, 128, F32, F32, 6)
    norm = module(4, 128, w, b)
    with torch.no_grad():
        y = norm(x.view(2, 40, 4, 128))
    want = osl.group_norm(x.reshape(80, 512).cpu(), 4, w.reshape(-1).cpu(), b.reshape(-1).cpu(), 1e-6).reshape(2, 40, 512)
    assert_parity(y.cpu(), torch.from_numpy(want), F32, "MultiHeadLayerNorm without a gradient")
