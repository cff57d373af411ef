"""The workspace of newton_schulz: asked for before the coefficients are known, it holds what any of them take."""

import pytest


@pytest.fixture(scope="module")
def lib():
    from xlstm_hip import _lib
    return _lib.load()


@pytest.mark.parametrize("batch,m,n", [(1, 200, 300), (3, 1000, 4000), (1, 64, 8000), (1, 128, 256), (12, 1024, 2048), (1, 65, 9000)])
def test_bfloat16_holds_the_pairs(lib, batch, m, n):
    """bfloat16 matrices run as pairs where the coefficients ask for it, as float16's do."""
    bf16, f16 = (lib.xl_newton_schulz_workspace_size(batch, m, n, dtype) for dtype in (1, 2))
    assert bf16 >= f16 > 0
    assert lib.xl_newton_schulz_workspace_size(batch, n, m, 1) == bf16


def test_small_matrices_need_none(lib):
    for m, n in ((1, 1), (64, 256), (128, 128), (256, 64)):
        assert all(lib.xl_newton_schulz_workspace_size(5, m, n, dtype) == 0 for dtype in (0, 1, 2))
