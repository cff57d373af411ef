"""The gated delta rule on the GPU where sizes are far apart: gradients beside a matrix of zeros.

Bars of gradients are those of test_gpu_gated_delta_bwd."""

import pytest
import torch

from test_gpu_gated_delta_bwd import check_all, inputs

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


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
