"""The layer norm's outputs that go past L2, in every layout of a row over lanes with one head and with several; and that
differentiating twice raises.

Bars as in test_gpu_layer_norm.py."""

import pytest
import torch

from helpers import dev
from test_gpu_layer_norm import BF16, F16, F32, check, inputs, reference

pytestmark = pytest.mark.gpu


# outputs of 16 MiB and more: every team size, one head and several, each with its last rows in a part of a workgroup
@pytest.mark.parametrize("tokens,H,D,dtype", [(66001, 1, 130, BF16), (4111, 8, 256, BF16), (9001, 4, 333, F16), (8195, 2, 512, BF16),
                                              (4099, 1, 2056, BF16), (2053, 1, 4096, BF16), (1027, 1, 8192, BF16),
                                              (517, 1, 16384, BF16), (1029, 4, 1024, F32), (263, 1, 16384, F32)])
def test_large_outputs(gpu_case, tokens, H, D, dtype):
    import xlstm_hip
    assert tokens * H * D * dtype.itemsize >= 16 << 20
    x, w, b, dy = inputs(tokens, H, D, dtype, F32, D)
    h, w1, b1 = (t.detach().requires_grad_(True) for t in (x.view(1, tokens, H, D), w.reshape(-1), b.reshape(-1)))
    y = xlstm_hip.multi_head_layer_norm(h, w1, b1, 1e-6, heads_first=False)
    dh, dw, db = torch.autograd.grad(y, (h, w1, b1), dy.view(1, tokens, H * D))
    got = (y.view(tokens, H, D), dh.view(tokens, H, D), dw.view(H, D), db.view(H, D))
    for a, (v, bar), name in zip(got, reference(x, w, b, dy, 1e-6), ("y", "dh", "dw", "db")):
        check(a, v, bar, name)


@pytest.mark.parametrize("call", ["layer_norm", "multi_head_layer_norm", "MultiHeadLayerNorm"])
def test_differentiating_twice_raises(gpu_case, call):
    """The first gradient keeps its history, and a backward through it raises."""
    import xlstm_hip
    x = torch.randn(2, 3, 4, 64, device=dev()).requires_grad_(True)
    run = {"layer_norm": xlstm_hip.layer_norm, "multi_head_layer_norm": xlstm_hip.multi_head_layer_norm,
           "MultiHeadLayerNorm": xlstm_hip.MultiHeadLayerNorm(4, 64).to(dev())}[call]
    (dx,) = torch.autograd.grad(run(x).square().sum(), x, create_graph=True)
    assert dx.requires_grad
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.square().sum(), x)
