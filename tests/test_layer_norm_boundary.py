"""The layer norm's boundary without a GPU: what the C entry points refuse before any GPU call, that CPU tensors
raise, and that a training step traces with symbolic sizes."""

import ctypes

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx


@pytest.fixture(scope="module")
def lib():
    from xlstm_hip import _lib
    return _lib.load()


P, Q, R = (ctypes.c_void_p(256 * (k + 1)) for k in range(3))  # never dereferenced: the checks fail first


def fwd(lib, x=P, y=Q, n=(1, 4), H=1, D=64, dtype=1, param=0):
    return lib.xl_layer_norm_fwd(x, None, None, None, y, None, None, *n, H, D, 1e-5, dtype, param, None)


def test_forward_refuses(lib):
    for bad in (dict(n=(-1, 4)), dict(n=(1, -4)), dict(H=0), dict(D=0), dict(dtype=5), dict(param=2), dict(dtype=0, param=1)):
        assert fwd(lib, **bad) == -1, bad
    assert fwd(lib, x=None) == -1 and b"null" in lib.xl_last_error()
    assert fwd(lib, y=P) == -1 and b"alias" in lib.xl_last_error()
    assert fwd(lib, n=(1 << 16, 1 << 16)) == -2
    assert fwd(lib, H=1 << 13, D=1 << 14) == -2
    assert fwd(lib, H=(1 << 20) + 1, D=1) == -2
    assert fwd(lib, n=(1 << 62, 1 << 62)) == -2
    assert fwd(lib, n=(0, 7)) == 0  # no rows


@pytest.mark.parametrize("eps", [-1e-6, float("nan"), float("inf")])
def test_forward_refuses_eps(lib, eps):
    """As the group norm does, which MultiHeadLayerNorm runs without a gradient."""
    assert lib.xl_layer_norm_fwd(P, None, None, None, Q, None, None, 1, 4, 1, 64, eps, 1, 0, None) == -1
    assert b"eps" in lib.xl_last_error()


def bwd(lib, dy=P, x=Q, mean=R, rstd=R, dx=None, dw=None, n=(1, 4), H=1, D=64, ws=None, ws_bytes=0):
    return lib.xl_layer_norm_bwd(dy, x, None, None, mean, rstd, dx, None, dw, None, *n, H, D, 1, 0, ws, ws_bytes, None)


def test_backward_refuses(lib):
    big = ctypes.c_void_p(4096)
    assert bwd(lib) == 0  # nothing asked for
    for bad in (dict(dy=None), dict(x=None), dict(mean=None), dict(rstd=None)):
        assert bwd(lib, dx=big, **bad) == -1 and b"null" in lib.xl_last_error()
    assert bwd(lib, dx=P) == -1 and bwd(lib, dx=Q) == -1
    assert bwd(lib, dx=big, D=0) == -1
    need = lib.xl_layer_norm_bwd_workspace_size(1, 4, 1, 64, 1)
    assert need > 0
    assert bwd(lib, dw=big) == -3 and b"workspace" in lib.xl_last_error()
    assert bwd(lib, dw=big, ws=big, ws_bytes=need - 1) == -3
    assert bwd(lib, dw=big, ws=ctypes.c_void_p(4100), ws_bytes=need) == -3
    assert lib.xl_layer_norm_bwd_workspace_size(1, 4, 1, 0, 1) == 0


def test_cpu_tensors_raise():
    import xlstm_hip
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        xlstm_hip.layer_norm(torch.randn(3, 8))
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        xlstm_hip.multi_head_layer_norm(torch.randn(1, 2, 3, 8))


@pytest.mark.parametrize("heads", [False, True])
def test_training_step_traces_with_symbolic_sizes(heads):
    import xlstm_hip

    def step(x, w, b):
        x, w, b = (t.detach().requires_grad_(True) for t in (x, w, b))
        y = xlstm_hip.multi_head_layer_norm(x, w, b) if heads else xlstm_hip.layer_norm(x, w, b)
        return torch.autograd.grad(y.sum(), (x, w, b))

    x = torch.randn(2, 3, 5, 64)
    w = torch.ones(192 if heads else 64)
    gm = make_fx(step, tracing_mode="symbolic")(x, w, w.clone())
    called = [str(n.target) for n in gm.graph.nodes if "xlstm_hip" in str(n.target)]
    assert called == ["xlstm_hip.layer_norm.default", "xlstm_hip.layer_norm_bwd.default"]
    out = [n for n in gm.graph.nodes if n.op == "output"][0].args[0]
    assert [tuple(o.meta["val"].shape) for o in out][1:] == [tuple(w.shape)] * 2
    q = next(n for n in gm.graph.nodes if n.op == "placeholder").meta["val"]
    assert not q.shape[2].node.expr.is_number
