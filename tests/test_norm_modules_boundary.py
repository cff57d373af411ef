"""MultiHeadLayerNorm's boundary without a GPU: what its kernel's entry point refuses, which operator a call traces to,
and with symbolic sizes."""

import ctypes

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

P, Q, R = (ctypes.c_void_p(256 * (k + 1)) for k in range(3))  # never dereferenced: the checks fail first


def test_statistics_come_together():
    from xlstm_hip import _lib
    lib = _lib.load()
    call = lambda **k: lib.xl_group_norm_stats_fwd(P, None, None, Q, k.get("mean"), k.get("rstd"), k.get("N", 4), 2, 64,  # noqa: E731
                                                   k.get("eps", 1e-6), k.get("dtype", 1), None)
    for one in (dict(mean=R), dict(rstd=R)):
        assert call(**one) == -1 and b"rstd" in lib.xl_last_error()
    for bad in (dict(N=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(dtype=7)):
        assert call(mean=R, rstd=P, **bad) == -1, bad
    assert call(mean=R, rstd=P, N=0) == 0


@pytest.mark.parametrize("dtype,param,grad,calls", [
    (torch.float32, torch.float32, True, ["layer_norm", "layer_norm_bwd"]), (torch.float32, torch.float32, False, ["group_norm"]),
    (torch.bfloat16, torch.float32, True, ["layer_norm", "layer_norm_bwd"]), (torch.bfloat16, torch.float32, False, ["layer_norm"])])
def test_traces_with_symbolic_sizes(dtype, param, grad, calls):
    import xlstm_hip
    norm = xlstm_hip.MultiHeadLayerNorm(4, 32, use_bias=True).to(param)

    def step(x):
        if not grad:
            with torch.no_grad():
                return norm(x)
        x = x.detach().requires_grad_(True)
        return torch.autograd.grad(norm(x).sum(), x)[0]

    gm = make_fx(step, tracing_mode="symbolic", _allow_non_fake_inputs=True)(torch.randn(2, 5, 4, 32).to(dtype))
    assert [str(n.target) for n in gm.graph.nodes if "xlstm_hip" in str(n.target)] == [f"xlstm_hip.{c}.default" for c in calls]
    out = [n for n in gm.graph.nodes if n.op == "output"][0].args[0].meta["val"]
    assert out.dtype == dtype and out.dim() == (4 if grad else 3) and not out.shape[1].node.expr.is_number


def test_cpu_tensors_raise():
    import xlstm_hip
    with pytest.raises(RuntimeError, match="must be on the GPU"):
        xlstm_hip.MultiHeadLayerNorm(4, 32)(torch.randn(2, 5, 4, 32))
