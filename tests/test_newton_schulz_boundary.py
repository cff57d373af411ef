"""The orthogonalisation's boundary without a GPU: what the C entry points refuse before any GPU call, the Python
checks, and tracing."""

import ctypes

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx


@pytest.fixture(scope="module")
def lib():
    from xlstm_hip import _lib
    return _lib.load()


P, Q, W = (ctypes.c_void_p(4096 * (k + 1)) for k in range(3))  # never dereferenced: the checks fail first


def call(lib, g=P, x=Q, batch=1, m=200, n=300, c=(3.4445, -4.775, 2.0315) * 5, steps=5, eps=1e-7, dtype=1, ws=W, ws_bytes=1 << 40):
    coefficients = None if c is None else (ctypes.c_float * len(c))(*c)
    return lib.xl_newton_schulz(g, x, batch, m, n, coefficients, steps, eps, dtype, ws, ws_bytes, None)


def test_refuses(lib):
    for bad in (dict(batch=-1), dict(m=-1), dict(n=-1), dict(dtype=4), dict(steps=0), dict(steps=65, c=(1.5, -0.5, 0.0) * 65), dict(c=None), dict(eps=-1e-9),
                dict(eps=float("nan")), dict(g=None), dict(x=None), dict(x=P)):
        assert call(lib, **bad) == -1, bad
    for bad in (dict(m=65537), dict(n=65537), dict(batch=65536)):
        assert call(lib, **bad) == -2, bad
    need = lib.xl_newton_schulz_workspace_size(1, 200, 300, 1)
    assert need > 0
    for bad in (dict(ws=None), dict(ws_bytes=need - 1), dict(ws=ctypes.c_void_p(4096 + 16))):
        assert call(lib, **bad) == -3 and b"workspace" in lib.xl_last_error(), bad
    assert lib.xl_newton_schulz_workspace_size(7, 64, 96, 1) == 0  # small matrices live in LDS
    for c in ((9.0, 0.0, 0.0), (3.0, 3.0, 3.0) * 2, (float("nan"), 0.0, 0.0), (1.0, float("inf"), 0.0), (0.0, -200.0, 200.0)):
        assert call(lib, c=c, steps=len(c) // 3) == -1 and b"out of range" in lib.xl_last_error(), c
    for empty in (dict(batch=0), dict(m=0), dict(n=0)):
        assert call(lib, **empty, g=None, x=None, ws=None, ws_bytes=0) == 0
        assert lib.xl_newton_schulz_workspace_size(empty.get("batch", 1), empty.get("m", 200), empty.get("n", 300), 1) == 0


def test_python_checks():
    import xlstm_hip
    x = torch.randn(4, 4)
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        xlstm_hip.newton_schulz(x)
    with pytest.raises(ValueError, match="steps"):
        xlstm_hip.newton_schulz(x, steps=0)
    with pytest.raises(ValueError, match="coefficients"):
        xlstm_hip.newton_schulz(x, 3, [(1.5, -0.5, 0.0)] * 2)
    with pytest.raises(ValueError, match="coefficients"):
        xlstm_hip.newton_schulz(x, 2, (1.5, -0.5))


def test_traces_with_symbolic_sizes():
    import xlstm_hip
    gm = make_fx(lambda x: xlstm_hip.newton_schulz(x * 2), tracing_mode="symbolic")(torch.randn(3, 20, 30))
    assert [str(n.target) for n in gm.graph.nodes if "xlstm_hip" in str(n.target)] == ["xlstm_hip.newton_schulz.default"]
    assert all(not d.node.expr.is_number for d in next(n for n in gm.graph.nodes if n.op == "placeholder").meta["val"].shape)
