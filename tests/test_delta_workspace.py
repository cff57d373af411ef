"""The workspace of the gated delta rule's gradients by the type of the gates, without a GPU: what the C entry point asks for and takes."""

import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from xlstm_hip import _lib
    return _lib.load()


SHAPE = (1, 2, 2, 100, 64, 64)
F32, BF16, F16 = 0, 1, 2
P, WS = ctypes.c_void_p(4096), ctypes.c_void_p(8192)  # never dereferenced: the strides are refused first


def backward(lib, dt, dg, bytes_):
    strides = (ctypes.c_int64 * 9)(64, 64, 64, 64, 64, 64, 64, 64, -1)
    return lib.xl_gated_delta_chunkwise_bwd(P, P, P, strides, P, P, None, P, None, P, P, P, P, P, None, *SHAPE, 0.1, dt, dg, WS, bytes_, None)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("dg", [F32, BF16, F16])
def test_size_by_the_gates(lib, dt, dg):
    need = lib.xl_gated_delta_chunkwise_bwd_workspace_size_gates(*SHAPE, dt, dg)
    most = lib.xl_gated_delta_chunkwise_bwd_workspace_size(*SHAPE, dt)
    assert (0 < need < most) if dt == dg == BF16 else need == most > 0
    assert backward(lib, dt, dg, need - 1) == -3 and b"workspace" in lib.xl_last_error()
    assert backward(lib, dt, dg, need) == -2 and b"strides" in lib.xl_last_error()


def test_refusals(lib):
    size = lib.xl_gated_delta_chunkwise_bwd_workspace_size_gates
    assert size(*SHAPE, BF16, 3) == 0 and size(*SHAPE, 5, F32) == 0
    assert size(1, 2, 2, 0, 64, 64, BF16, F32) == 0
