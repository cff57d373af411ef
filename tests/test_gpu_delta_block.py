"""The gated delta rule, the norms and the gated linear unit together, as a model's block: trained, prefilled and decoded, eagerly and
in captured graphs; and the stack with its feed-forward block in one kernel.

Bars of the block's outputs and gradients, bf16: along the longest path at most 16 values are rounded to bf16 one after another (norm,
projection, q / k norm, mixer, its operands, head norm, projection, sum; norm, unit, its factors, projection, sum; and back), each
by 2^-9 of itself at most: 16 2^-9 = 3.2e-2 of the norm, were they all of one sign."""

import pytest
import torch
import torch.nn.functional as F

from helpers import dev

pytestmark = pytest.mark.gpu
BAR = 16 * 2.0 ** -9
D, NH, NHK, DQK, DV, FF = 128, 4, 2, 32, 48, 200


def weights(seed=0, dtype=torch.bfloat16):
    r = torch.Generator().manual_seed(seed)
    n = lambda *s: (torch.randn(*s, generator=r) * s[-1] ** -0.5).to(dtype).to(dev())  # noqa: E731
    return dict(n1=torch.ones(D, dtype=dtype, device=dev()), q=n(NHK * DQK, D), k=n(NHK * DQK, D), v=n(NH * DV, D), gates=n(2 * NH, D),
                hw=torch.ones(NH * DV, dtype=dtype, device=dev()), out=n(D, NH * DV), n2=torch.ones(D, dtype=dtype, device=dev()),
                wg=n(FF, D), wu=n(FF, D), down=n(D, FF))


def heads(x, w, n):
    B, S, _ = x.shape
    return F.linear(x, w).view(B, S, n, -1).transpose(1, 2)


def mixer_inputs(y, w):
    q, k, v = (heads(y, w[m], n) for m, n in (("q", NHK), ("k", NHK), ("v", NH)))
    q, k = (F.normalize(t.float() if t.dtype != torch.float64 else t, dim=-1).to(t.dtype) for t in (q, k))
    g, beta = heads(y, w["gates"], 2 * NH).squeeze(-1).chunk(2, 1)
    return q, k, v, -0.1 * F.softplus(g), torch.sigmoid(beta)


def block(x, w, ops, c0=None):
    """(x', the mixer's state); ops: layer norm, mixer, head norm, unit."""
    norm, mixer, head_norm, unit = ops
    h, c = mixer(*mixer_inputs(norm(x, w["n1"]), w), c0)
    x = x + F.linear(head_norm(h, w["hw"]), w["out"])
    return x + F.linear(unit(norm(x, w["n2"]), w["wg"], w["wu"]), w["down"]), c


def hip_ops(mixer=None):
    import xlstm_hip
    mixer = mixer or xlstm_hip.gated_delta_chunkwise
    return (lambda x, w: xlstm_hip.layer_norm(x, w), lambda *a: mixer(*a, return_last_states=True),
            lambda h, w: xlstm_hip.multi_head_layer_norm(h, w), xlstm_hip.gated_linear_unit)


def plain_mixer(q, k, v, g, beta, c0):
    rep = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    C, h = (v.new_zeros(*v.shape[:2], q.shape[-1], v.shape[-1]) if c0 is None else c0), []
    for t in range(v.shape[2]):
        C = C * torch.exp(g[:, :, t, None, None])
        d = beta[:, :, t, None] * (v[:, :, t] - (k[:, :, t, :, None] * C).sum(-2))
        C = C + k[:, :, t, :, None] * d[..., None, :]
        h.append(q.shape[-1] ** -0.5 * (q[:, :, t, :, None] * C).sum(-2))
    return torch.stack(h, 2), C


PLAIN = (lambda x, w: F.layer_norm(x, (x.shape[-1],), w), plain_mixer,
         lambda h, w: (F.layer_norm(h.transpose(1, 2), (DV,), eps=1e-6).flatten(2) * w),
         lambda x, wg, wu: F.silu(F.linear(x, wg)) * F.linear(x, wu))


def tokens(B, S, seed=1):
    return torch.randn(B, S, D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(dev())


def off(a, b):
    return float((a.double() - b).norm() / b.norm())


def test_training_step(gpu_case):
    x, w, dy = tokens(2, 100), weights(), tokens(2, 100, 2)
    leaves = lambda cast: [cast(t).detach().requires_grad_(True) for t in (x, *w.values())]  # noqa: E731
    got, want = leaves(lambda t: t), leaves(lambda t: t.double())
    y, _ = block(got[0], dict(zip(w, got[1:])), hip_ops())
    yr, _ = block(want[0], dict(zip(w, want[1:])), PLAIN)
    assert off(y, yr) <= BAR
    for a, b, name in zip(torch.autograd.grad(y, got, dy), torch.autograd.grad(yr, want, dy.double()), ("x", *w)):
        assert off(a, b) <= BAR, name


def test_prefill_then_decode(gpu_case):
    """A prompt by chunks, drafted tokens by the recurrent kernel, then steps in place: the whole sequence's outputs."""
    import xlstm_hip
    x, w = tokens(3, 90), weights()
    with torch.no_grad():
        want, last = block(x.double(), {n: t.double() for n, t in w.items()}, PLAIN)
        y, c = block(x[:, :70], w, hip_ops())
        parts = [y]
        y, c = block(x[:, 70:80], w, hip_ops(xlstm_hip.gated_delta_recurrent), c)
        parts.append(y)

        def step(*a):
            h, s = xlstm_hip.gated_delta_step_(*(t[:, :, 0] for t in a[:5]), a[5])
            return h[:, :, None], s

        ops = list(hip_ops())
        ops[1] = step
        for t in range(80, 90):
            y, c = block(x[:, t:t + 1], w, ops, c)
            parts.append(y)
        got = torch.cat(parts, 1)
    for t in range(90):
        assert off(got[:, t], want[:, t]) <= BAR, t
    assert off(c, last) <= BAR


def captured(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def check_replays(fn, inputs, change):
    """Replays on changing inputs, each against the eager call, with eager work and synchronisation between."""
    graph, out = captured(fn)
    for r in range(4):
        change(r)
        kept = [t.clone() for t in inputs]
        want = [t.clone() for t in fn()]
        for t, k in zip(inputs, kept):
            t.copy_(k)
        torch.randn(1 << 16, device=dev()).sum()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), r


def test_captured_decode(gpu_case):
    import xlstm_hip
    x, w = tokens(2, 1), weights()
    c = torch.randn(2, NH, DQK, DV, device=dev())

    def step(*a):
        h, s = xlstm_hip.gated_delta_step_(*(t[:, :, 0] for t in a[:5]), a[5])
        return h[:, :, None], s

    ops = list(hip_ops())
    ops[1] = step

    def fn():
        with torch.no_grad():
            return block(x, w, ops, c)

    check_replays(fn, [x, c], lambda r: (x.copy_(tokens(2, 1, 10 + r)), c.normal_()))


@pytest.mark.parametrize("state", [False, True])
def test_captured_training_step(gpu_case, state):
    x, w, dy = tokens(2, 100), weights(), tokens(2, 100, 2)
    c0 = torch.randn(2, NH, DQK, DV, device=dev()) if state else None
    leaves = [t.detach().requires_grad_(True) for t in (x, *w.values())]

    def fn():
        y, c = block(leaves[0], dict(zip(w, leaves[1:])), hip_ops(), c0)
        return [y.detach(), *torch.autograd.grad([y, c] if state else [y], leaves, [dy, torch.ones_like(c)] if state else [dy])]

    def change(r):
        with torch.no_grad():
            leaves[0].copy_(tokens(2, 100, 20 + r))

    check_replays(fn, [], change)


def test_two_captured_at_once(gpu_case):
    """Two graphs of the same operators, replayed on two streams at a time: nothing between them is shared."""
    xs = [tokens(2, 200, s) for s in (1, 2)]
    w = weights()
    fns = [lambda x=x: block(x, w, hip_ops()) for x in xs]
    with torch.no_grad():
        want = [[t.clone() for t in f()] for f in fns]
        graphs = [captured(f) for f in fns]
        streams = [torch.cuda.Stream() for _ in fns]
        for _ in range(3):
            for (g, _), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            for (_, out), ref in zip(graphs, want):
                assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_stack_with_the_fused_block(gpu_case):
    """A small stack's logits with and without it: each block's feed-forward result moves by its roundings alone (three of 2^-9 of
    itself at most, of two blocks, behind them the final norm and the logits' own two): 8 2^-9 of the logits' norm."""
    import dataclasses
    from xlstm_hip.stack import StackConfig, xLSTMStack
    cfg = StackConfig("small", d_model=256, num_blocks=2, mlstm_heads=2, vocab=512)
    plain = xLSTMStack.random(cfg, dev(), seed=3)
    fused = xLSTMStack.random(dataclasses.replace(cfg, fused_ffn=True), dev(), seed=3)
    prompt = torch.randint(512, (2, 70), generator=torch.Generator().manual_seed(1)).to(dev())
    a, sa = plain.prefill(prompt)
    b, sb = fused.prefill(prompt)
    assert off(b, a.double()) <= 8 * 2.0 ** -9
    token = a.argmax(-1)
    a, b = plain.decode_step(token, sa), fused.decode_step(token, sb)
    assert off(b, a.double()) <= 8 * 2.0 ** -9
    assert torch.equal(fused.generate(prompt, 6, graph=True), fused.generate(prompt, 6, graph=False))


def test_fused_block_differentiates(gpu_case):
    from xlstm_hip.stack import _FFN
    ffn = _FFN(128, 200, fused=True).to(torch.bfloat16).to(dev())
    x = tokens(2, 50).requires_grad_(True)
    ffn(x).sum().backward()
    want = [t.grad.clone() for t in (x, *ffn.parameters())]
    ref = _FFN(128, 200).double().to(dev())
    ref.load_state_dict(ffn.state_dict())
    y = x.detach().double().requires_grad_(True)
    ref(y).sum().backward()
    for a, b in zip(want, (y, *ref.parameters())):
        assert off(a, b.grad) <= 6 * 2.0 ** -9
