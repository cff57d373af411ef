"""Calls of the gated delta rule at the edges of their shapes: one token under any stride, an empty batch."""

import pytest
import torch

from delta_reference import make
from helpers import dev

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def test_one_token_under_any_stride(gpu_case):
    """A slice of one token of [S, B, NH, D] tensors: its token stride is B NH D, above 2^22, and never stepped."""
    import xlstm_hip
    x = make(2, 2, 2, 1, 64, 48, BF16, F32, seed=1)

    def far(t):
        y = torch.as_strided(torch.empty(4096, dtype=t.dtype, device=dev()), t.shape, (2 * t.shape[-1], t.shape[-1], 1 << 33, 1))
        return y.copy_(t)

    y = [far(t) for t in x[:3]] + list(x[3:])
    assert y[0].stride(2) == 1 << 33
    for op in (xlstm_hip.gated_delta_chunkwise, xlstm_hip.gated_delta_recurrent):
        for a, b in zip(op(*y, return_last_states=True), op(*x, return_last_states=True)):
            assert torch.equal(a, b)
    found = []
    for z in (x, y):
        z = [t.detach().requires_grad_(True) for t in z]
        h, c = xlstm_hip.gated_delta_chunkwise(*z, return_last_states=True)
        found.append(torch.autograd.grad(h.float().sum() + c.sum(), z))
    assert all(torch.equal(a, b) for a, b in zip(*found))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_empty_batch(gpu_case, dtype):
    """No sequences: empty results and gradients, as without tokens."""
    import xlstm_hip
    x = [t[:0] for t in make(1, 4, 2, 70, 64, 48, dtype, F32, seed=2)]
    for op in (xlstm_hip.gated_delta_chunkwise, xlstm_hip.gated_delta_recurrent):
        h, c = op(*x, return_last_states=True)
        assert h.shape == (0, 4, 70, 48) and h.dtype == dtype and c.shape == (0, 4, 64, 48) and c.dtype == F32
        assert op(*x[:5]).shape == (0, 4, 70, 48)
    one = [t[:, :, 0] for t in x[:5]]
    h, c = xlstm_hip.gated_delta_step(*one, x[5])
    assert h.shape == (0, 4, 48) and c.shape == (0, 4, 64, 48)
    h, c = xlstm_hip.gated_delta_step_(*one, x[5])
    assert h.shape == (0, 4, 48) and c is x[5]
    y = [t.detach().requires_grad_(True) for t in x]
    h, c = xlstm_hip.gated_delta_chunkwise(*y, return_last_states=True)
    for g, t in zip(torch.autograd.grad((h, c), y, (torch.ones_like(h), torch.ones_like(c))), y):
        assert g.shape == t.shape and g.dtype == t.dtype
