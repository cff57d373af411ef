"""The gated delta rule's and the gated linear unit's boundary without a GPU: what the C entry points refuse before any GPU call,
what the operators refuse, and that training steps trace with symbolic sizes."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx


@pytest.fixture(scope="module")
def lib():
    from xlstm_hip import _lib
    return _lib.load()


P, Q, WS = (ctypes.c_void_p(4096 * (k + 1)) for k in range(3))  # never dereferenced: the checks fail first
I64x9 = ctypes.c_int64 * 9


def delta(lib, which="chunkwise_fwd", q=P, h=Q, c0=None, cl=None, B=1, NH=2, NHK=2, S=100, DQK=64, DV=64, dt=1, dg=0, ws=None, n=0, strides=None):
    if which == "recurrent_fwd":
        return lib.xl_gated_delta_recurrent_fwd(q, P, P, P, P, c0, h, cl, B, NH, NHK, S, DQK, DV, 0.1, dt, dg, None)
    if which == "chunkwise_fwd":
        return lib.xl_gated_delta_chunkwise_fwd(q, P, P, strides, P, P, c0, h, cl, B, NH, NHK, S, DQK, DV, 0.1, dt, dg, ws, n, None)
    return lib.xl_gated_delta_chunkwise_bwd(q, P, P, strides, P, P, c0, P, cl, h, P, P, P, P, c0, B, NH, NHK, S, DQK, DV, 0.1, dt, dg, ws, n, None)


@pytest.mark.parametrize("which", ["recurrent_fwd", "chunkwise_fwd", "chunkwise_bwd"])
def test_delta_refuses(lib, which):
    for bad in (dict(B=0), dict(NH=0), dict(NHK=0), dict(S=-1), dict(DQK=0), dict(DV=0), dict(NH=3), dict(dt=5), dict(dg=3)):
        assert delta(lib, which, **bad) == -1, bad
    assert delta(lib, which, DQK=257) == -2 and b"DQK" in lib.xl_last_error()
    assert delta(lib, which, B=1 << 20, NH=1 << 10, NHK=1) == -2
    assert delta(lib, which, B=1 << 10, NH=1 << 10, NHK=1, S=1 << 20, DV=512) == -2
    assert delta(lib, which, q=None) == -1 and b"null" in lib.xl_last_error()
    assert delta(lib, which, h=None) == -1
    if which != "recurrent_fwd":
        need = getattr(lib, f"xl_gated_delta_{which.replace('_fwd', '')}_workspace_size")(1, 2, 2, 100, 64, 64, 1)
        assert need > 0
        assert delta(lib, which) == -3 and b"workspace" in lib.xl_last_error()
        assert delta(lib, which, ws=WS, n=need - 1) == -3
        assert delta(lib, which, ws=ctypes.c_void_p(4096 + 16), n=need) == -3
        assert delta(lib, which, h=ctypes.c_void_p(4096 + 8), ws=WS, n=need) == -1 and b"aligned" in lib.xl_last_error()
        assert delta(lib, which, c0=P, cl=P, ws=WS, n=need) == -1 and b"alias" in lib.xl_last_error()
        for step in (-1, 1 << 23):
            assert delta(lib, which, ws=WS, n=need, strides=I64x9(64, 64, 64, 64, 64, 64, 64, 64, step)) == -2
    if which == "chunkwise_bwd":
        assert delta(lib, which, S=0) == -1
    else:
        assert delta(lib, which, S=0, q=None, h=None) == 0  # nothing to do


@pytest.mark.parametrize("which", ["recurrent_fwd", "chunkwise_fwd", "chunkwise_bwd"])
def test_delta_refuses_more_threads_than_a_launch_has(lib, which):
    assert delta(lib, which, B=1 << 19, NH=1, NHK=1, S=1, DQK=1, DV=1024) == -2 and b"too large" in lib.xl_last_error()
    assert delta(lib, which, B=(1 << 24) - 1, NH=1, NHK=1, S=1, DQK=1, DV=33) == -2


def test_delta_workspace_sizes(lib):
    fwd, bwd = lib.xl_gated_delta_chunkwise_workspace_size, lib.xl_gated_delta_chunkwise_bwd_workspace_size
    assert fwd(1, 2, 2, 0, 64, 64, 1) == bwd(1, 2, 2, 0, 64, 64, 1) == 0
    assert fwd(1, 2, 2, 64, 300, 64, 1) == bwd(1, 2, 3, 64, 64, 64, 1) == 0  # refused
    assert fwd(1, 2, 2, 64, 64, 64, 1) < fwd(1, 2, 2, 65, 64, 64, 1) == fwd(1, 2, 2, 128, 64, 64, 1)
    # beyond 32 bits: 16 heads of 256 x 512 over half a million tokens
    assert bwd(1, 16, 16, 1 << 19, 256, 512, 0) > 1 << 37


def glu(lib, x=P, h=Q, a=None, u=None, pitch=0, T=4, D=64, F=40, act=0, dt=1, ws=None, n=0):
    return lib.xl_gated_linear_fwd(x, P, P, h, a, u, pitch, T, D, F, act, dt, ws, n, None)


def glu_bwd(lib, dh=P, a=P, u=P, pitch=40, dx=Q, dwg=Q, dwu=Q, T=4, D=64, F=40, act=0, dt=1, ws=None, n=0):
    return lib.xl_gated_linear_bwd(dh, P, P, P, a, u, pitch, dx, dwg, dwu, T, D, F, act, dt, ws, n, None)


def test_linear_refuses(lib):
    for call in (glu, glu_bwd):
        for bad in (dict(T=-1), dict(D=0), dict(F=0), dict(act=2), dict(dt=7)):
            assert call(lib, **bad) == -1, bad
        assert call(lib, dt=0) == -2 and b"float32" in lib.xl_last_error()
        assert call(lib, T=1 << 30) == -2
    assert glu(lib, x=None) == -1 and glu(lib, h=None) == -1 and b"null" in lib.xl_last_error()
    assert glu(lib, a=P) == -1 and b"together" in lib.xl_last_error()
    for pitch in (32, 44):
        assert glu(lib, a=P, u=P, pitch=pitch) == -1 and b"keep_pitch" in lib.xl_last_error()
        assert glu_bwd(lib, pitch=pitch) == -1
    assert glu(lib, x=ctypes.c_void_p(4098)) == -1 and b"aligned" in lib.xl_last_error()
    assert glu(lib, D=33) == -3 and b"workspace" in lib.xl_last_error()
    assert glu(lib, T=0, x=None) == 0
    assert glu_bwd(lib, dx=None, dwg=None, dwu=None) == 0  # nothing asked for
    assert glu_bwd(lib, dwg=None) == -1 and b"together" in lib.xl_last_error()
    assert glu_bwd(lib, T=0) == -1
    assert glu_bwd(lib, dh=None) == -1
    need = lib.xl_gated_linear_workspace_size(4, 64, 40, 1, 1)
    assert need >= 2 * 64 * 64 * 2
    assert glu_bwd(lib) == -3 and glu_bwd(lib, ws=WS, n=need - 1) == -3
    assert lib.xl_gated_linear_workspace_size(4, 64, 40, 0, 1) == 0  # rows of whole 16 bytes need none
    assert lib.xl_gated_linear_workspace_size(4, 0, 40, 0, 1) == 0


def x_delta(dt=torch.bfloat16, S=70, **kw):
    s = (2, 2, S) if S else (2, 2)
    v = (2, 4, S) if S else (2, 4)
    return [torch.randn(*s, 64, dtype=dt, **kw), torch.randn(*s, 64, dtype=dt, **kw), torch.randn(*v, 48, dtype=dt, **kw),
            torch.randn(*v, **kw), torch.randn(*v, **kw)]


def test_cpu_tensors_raise():
    import xlstm_hip
    for op, x in ((xlstm_hip.gated_delta_chunkwise, x_delta()), (xlstm_hip.gated_delta_recurrent, x_delta()),
                  (xlstm_hip.gated_delta_step, x_delta(S=0) + [torch.zeros(2, 4, 64, 48)]),
                  (xlstm_hip.gated_delta_step_, x_delta(S=0) + [torch.zeros(2, 4, 64, 48)]),
                  (xlstm_hip.gated_linear_unit, [torch.randn(3, 8)] * 3)):
        with pytest.raises(RuntimeError, match="must be on the GPU"):
            op(*x)


def test_unknown_activation():
    import xlstm_hip
    with pytest.raises(ValueError, match="activation"):
        xlstm_hip.gated_linear_unit(torch.randn(3, 8), torch.randn(4, 8), torch.randn(4, 8), "tanh")


@pytest.mark.parametrize("state", [False, True])
def test_delta_training_step_traces_with_symbolic_sizes(state):
    import xlstm_hip
    x = x_delta() + ([torch.randn(2, 4, 64, 48)] if state else [])

    def step(*x):
        x = [t.detach().requires_grad_(True) for t in x]
        h, c = xlstm_hip.gated_delta_chunkwise(*x, return_last_states=True)
        return torch.autograd.grad(h.sum() + c.sum(), x)

    gm = make_fx(step, tracing_mode="symbolic")(*x)
    called = [str(n.target) for n in gm.graph.nodes if "xlstm_hip" in str(n.target)]
    assert called == ["xlstm_hip.gated_delta_chunkwise.default", "xlstm_hip.gated_delta_chunkwise_bwd.default"]
    q = next(n for n in gm.graph.nodes if n.op == "placeholder").meta["val"]
    assert not q.shape[2].node.expr.is_number
    out = [n for n in gm.graph.nodes if n.op == "output"][0].args[0]
    assert [o.meta["val"].dtype for o in out] == [t.dtype for t in x]


def test_linear_training_step_traces_with_symbolic_sizes():
    import xlstm_hip
    x = [torch.randn(2, 30, 64, dtype=torch.bfloat16), *(torch.randn(43, 64, dtype=torch.bfloat16) for _ in range(2))]

    def step(*x):
        x = [t.detach().requires_grad_(True) for t in x]
        return torch.autograd.grad(xlstm_hip.gated_linear_unit(*x).sum(), x)

    gm = make_fx(step, tracing_mode="symbolic")(*x)
    called = [str(n.target) for n in gm.graph.nodes if "xlstm_hip" in str(n.target)]
    assert called == ["xlstm_hip.gated_linear.default", "xlstm_hip.gated_linear_bwd.default"]
    q = next(n for n in gm.graph.nodes if n.op == "placeholder").meta["val"]
    assert all(not d.node.expr.is_number for d in q.shape)


def test_in_place_step_moves_the_version_counter():
    import xlstm_hip
    with FakeTensorMode():
        x, c = x_delta(S=0, device="cuda"), torch.zeros(2, 4, 64, 48, device="cuda")
        h, back = xlstm_hip.gated_delta_step_(*x, c)
        assert back is c and c._version == 1 and h.shape == (2, 4, 48)
        x[2].requires_grad_(True)
        h, _ = xlstm_hip.gated_delta_step_(*x, c)
        with pytest.raises(RuntimeError):
            h.grad_fn(torch.ones_like(h))
