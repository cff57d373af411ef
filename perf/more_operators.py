"""Performance cases of the block operators beside the mLSTM: the gated delta rule (chunkwise with its backward pass,
token by token, and one decode step) and the gated linear unit of a feed-forward block with its backward pass.

A case is a dict of plain values; ``kind`` names the call:

* ``chunk``  ``gated_delta_chunkwise`` over [B, NH, S]; q and k have ``NHK`` heads, each shared by NH / NHK of v's
* ``short``  ``gated_delta_recurrent`` over a few tokens from a state
* ``step``   ``gated_delta_step``, one token from a state
* ``glu``    ``gated_linear_unit`` of ``T`` tokens: silu(x Wg^T) * (x Wu^T), weights [F, D]

``train`` adds the backward pass; ``state`` an initial state and the last one (with its gradient where ``train``);
``gate`` is the type of the gates g (log decay) and beta.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ESZ = {"bf16": 2, "f16": 2, "f32": 4}
CHUNK = 64

_hip = None


def _framework():
    """The package, imported once and only where its kernels run."""
    global _hip
    if _hip is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xlstm-metal_amd"))
        import xlstm_hip
        _hip = xlstm_hip
    return _hip


# ------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # serving one sequence at the smaller model's heads: one token (latency)
        dict(name="step_one", kind="step", B=1, NH=8, NHK=8, DQK=128, DV=256, dtype="bf16", gate="bf16"),
        # decoding a batch of 16 at the 7B model's heads (a stream through the state)
        dict(name="step_batch", kind="step", B=16, NH=8, NHK=8, DQK=256, DV=512, dtype="bf16", gate="f32"),
        # a few drafted tokens checked for each of 4 sequences
        dict(name="short_draft", kind="short", B=4, NH=8, NHK=8, S=13, DQK=128, DV=256, dtype="bf16", gate="bf16"),
        # one prompt of a ragged length, from and to a state, at the smaller model's heads
        dict(name="chunk_prompt", kind="chunk", B=1, NH=8, NHK=8, S=777, DQK=128, DV=256, dtype="bf16", gate="f32",
             state=True, train=False),
        # prefill of 4 long prompts at the 7B model's heads
        dict(name="chunk_prefill", kind="chunk", B=4, NH=8, NHK=8, S=8192, DQK=256, DV=512, dtype="bf16", gate="bf16",
             state=False, train=False),
        # training of the smaller model: 8192 tokens
        dict(name="chunk_train", kind="chunk", B=2, NH=8, NHK=8, S=4096, DQK=128, DV=256, dtype="bf16", gate="bf16",
             state=False, train=True),
        # float32 training through carried states, two heads of v to each of q and k, odd sizes
        dict(name="chunk_train_f32", kind="chunk", B=2, NH=4, NHK=2, S=501, DQK=100, DV=200, dtype="f32", gate="f32",
             state=True, train=True),
        # decoding 8 sequences through the 7B model's feed-forward block (a stream through the weights)
        dict(name="glu_token", kind="glu", T=8, D=4096, F=10944, dtype="bf16", train=False),
        # the ragged prompt through the smaller model's block
        dict(name="glu_prompt", kind="glu", T=777, D=2048, F=5504, dtype="bf16", train=False),
        # a long prompt through the 7B model's block
        dict(name="glu_prefill", kind="glu", T=8192, D=4096, F=10944, dtype="bf16", train=False),
        # training of the 7B model's block: 8192 tokens
        dict(name="glu_train", kind="glu", T=8192, D=4096, F=10944, dtype="bf16", train=True),
        # training at sizes that no tile divides
        dict(name="glu_train_odd", kind="glu", T=1333, D=1000, F=2731, dtype="f16", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("chunk", "chunk", "chunk", "short", "step", "glu", "glu", "glu"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    if kind == "glu":
        train = rng.random() < 0.5
        return dict(kind=kind, T=_log(rng, 1, 8192), D=_log(rng, 64, 4096), F=_log(rng, 64, 10944), dtype=dtype, train=train)
    dtype = rng.choice((dtype, dtype, "f32"))
    NHK, shared = rng.choice((1, 2, 4, 8)), rng.choice((1, 1, 1, 2, 3))
    DQK, DV = rng.choice((32, 64, 72, 96, 128, 192, 256)), rng.choice((32, 64, 100, 128, 200, 256, 512))
    case = dict(kind=kind, NH=NHK * shared, NHK=NHK, DQK=DQK, DV=DV, dtype=dtype)
    if kind == "step":
        return dict(case, B=_log(rng, 1, 32 // shared), gate=rng.choice((dtype, "f32")))
    if kind == "short":
        return dict(case, B=rng.choice((1, 2, 4)), S=rng.randint(2, 40), gate=rng.choice((dtype, "f32")))
    train = rng.random() < 0.4
    B = rng.choice((1, 1, 2, 4))
    return dict(case, B=B, S=_log(rng, 1, min(8192, 262144 // (B * case["NH"])) if not train else 2048 // B), gate=dtype if train else rng.choice((dtype, "f32")),
                state=rng.random() < 0.5 and (dtype == "f32" or not train), train=train)


# ------------------------------------------------------------------------------------- inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _inputs(case, seed):
    r = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DT[case["dtype"]]
    if case["kind"] == "glu":
        T, D, F = case["T"], case["D"], case["F"]
        # activations behind a norm, weights that give gate and up values of about 1
        x, wg, wu = (_randn(r, *s).mul_(f).to(dt) for s, f in (((T, D), 1.0), ((F, D), D ** -0.5), ((F, D), D ** -0.5)))
        return x, wg, wu, _randn(r, T, F).mul_(0.1).to(dt) if case["train"] else None
    B, NH, NHK, DQK, DV = (case[n] for n in ("B", "NH", "NHK", "DQK", "DV"))
    lead = () if case["kind"] == "step" else (case["S"],)
    # queries and keys of length 1, as the models norm them; keys drift, so that neighbours are alike
    q, k = _randn(r, B, NHK, *lead, DQK), _randn(r, B, NHK, *lead, DQK) + 0.5 * _randn(r, B, NHK, *((1,) * len(lead)), DQK)
    q, k = (t / t.norm(dim=-1, keepdim=True) for t in (q, k))
    v = _randn(r, B, NH, *lead, DV)
    # a head's time constant from a few tokens to thousands, as exp(A) softplus(.) spreads them
    g = -torch.exp(-7.0 * _rand(r, B, NH, *((1,) * len(lead)))) * torch.nn.functional.softplus(_randn(r, B, NH, *lead))
    beta = torch.sigmoid(_randn(r, B, NH, *lead))
    gt = DT[case["gate"]]
    c0 = 0.3 * _randn(r, B, NH, DQK, DV) if case["kind"] != "chunk" or case["state"] else None
    dh = dc = None
    if case.get("train"):
        dh = _randn(r, B, NH, *lead, DV).to(dt)
        dc = 0.1 * _randn(r, B, NH, DQK, DV) if case["state"] else None
    return (q.to(dt), k.to(dt), v.to(dt), g.to(gt), beta.to(gt), c0), dh, dc


def prepare(case, seed):
    state = dict(case=case, inputs=_inputs(case, seed))
    if case.get("train"):
        for t in state["inputs"][:3] if case["kind"] == "glu" else state["inputs"][0]:
            if t is not None:
                t.requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["kind"] == "glu":
        x, wg, wu, dh = state["inputs"]
        if not own:
            with torch.no_grad():
                return _plain_glu(x, wg, wu, dh)
        h = _framework().gated_linear_unit(x, wg, wu)
        return (h.detach(), *torch.autograd.grad(h, (x, wg, wu), dh)) if case["train"] else h
    if case["kind"] == "step":
        q, k, v, g, beta, c0 = state["inputs"][0]
        return _framework().gated_delta_step(q, k, v, g, beta, c0) if own else _plain_step(q, k, v, g, beta, c0)
    given, dh, dc = state["inputs"]
    if case["kind"] == "short":
        if own:
            return _framework().gated_delta_recurrent(*given, return_last_states=True)
        return _plain_delta(*given)
    if own:
        h = _framework().gated_delta_chunkwise(*given, return_last_states=case["state"])
        h, c = h if case["state"] else (h, None)
    else:
        h, c = _plain_delta(*given)
    if not case["train"]:
        return (h, c) if case["state"] else h
    leaves = [t for t in given if t is not None]
    if case["state"]:
        return (h.detach(), c.detach(), *torch.autograd.grad((h, c), leaves, (dh, dc)))
    return (h.detach(), *torch.autograd.grad(h, leaves, dh))


def _plain_glu(x, wg, wu, dh):
    xf, gf, uf = x.float(), wg.float(), wu.float()
    a, u = torch.matmul(xf, gf.t()), torch.matmul(xf, uf.t())
    s = 1.0 / (1.0 + torch.exp(-a))
    h = (a * s * u).to(x.dtype)
    if dh is None:
        return h
    d = dh.float()
    da, du = d * u * (s * (1.0 + a * (1.0 - s))), d * (a * s)
    dx = torch.matmul(da, gf) + torch.matmul(du, uf)
    return h, dx.to(x.dtype), torch.matmul(da.t(), xf).to(wg.dtype), torch.matmul(du.t(), xf).to(wu.dtype)


def _plain_step(q, k, v, g, beta, c0):
    """a = exp(g); d = beta (v - a C^T k); C' = a C + k d^T; h = C'^T q / sqrt(DQK)."""
    shared = v.shape[1] // q.shape[1]
    qf, kf = (t.float().repeat_interleave(shared, 1) for t in (q, k))
    c = c0 * torch.exp(g.float())[..., None, None]
    d = beta.float()[..., None] * (v.float() - (c * kf[..., None]).sum(-2))
    c = c + kf[..., None] * d[..., None, :]
    return ((c * qf[..., None]).sum(-2) * q.shape[-1] ** -0.5).to(v.dtype), c


def _plain_delta(q, k, v, g, beta, c0):
    """The recurrence of _plain_step by chunks of 64 tokens: within a chunk the corrections d solve (I + A) D = beta (V -
    decayed K C), A below the diagonal, whose inverse is a product of six factors (in 64 bits: its powers grow).  The one
    loop is over the chunks, each of which starts from the state of the one before."""
    S, scale, shared = q.shape[2], q.shape[-1] ** -0.5, v.shape[1] // q.shape[1]
    L = min(CHUNK, S)
    pad = -S % L

    def chunks(t, heads):
        t = t.float()
        if pad:
            t = torch.cat([t, t.new_zeros(t.shape[:2] + (pad,) + t.shape[3:])], 2)
        t = t if heads == 1 else t.repeat_interleave(heads, 1)
        return t.reshape(t.shape[:2] + (-1, L) + t.shape[3:])

    qc, kc, vc, gc, bc = chunks(q, shared), chunks(k, shared), chunks(v, 1), chunks(g, 1), chunks(beta, 1)
    i = torch.arange(L, device=q.device)
    low, strict = i[:, None] >= i[None, :], i[:, None] > i[None, :]
    b = gc.double().cumsum(-1)
    decay = torch.exp((b[..., :, None] - b[..., None, :]).masked_fill(~low, -math.inf)).float()
    A = (bc[..., None] * decay * torch.matmul(kc, kc.transpose(-1, -2)) * strict).double()
    eye = torch.eye(L, dtype=torch.float64, device=q.device)
    A2 = torch.matmul(A, A)
    A4 = torch.matmul(A2, A2)
    A8 = torch.matmul(A4, A4)
    A16 = torch.matmul(A8, A8)
    A32 = torch.matmul(A16, A16)
    inv = torch.matmul(torch.matmul(torch.matmul(eye - A, eye + A2), torch.matmul(eye + A4, eye + A8)),
                       torch.matmul(eye + A16, eye + A32))
    inv = (inv * bc[..., None, :]).float()
    c_in = torch.exp(b).float()[..., None]
    c_out = torch.exp(b[..., -1:] - b).float()[..., None]
    c_all = torch.exp(b[..., -1]).float()[..., None, None]
    U, W = torch.matmul(inv, vc), torch.matmul(inv, c_in * kc)
    P = torch.matmul(qc, kc.transpose(-1, -2)) * decay * scale
    qd, kd = qc * c_in * scale, (kc * c_out).transpose(-1, -2)
    C = c0 if c0 is not None else torch.zeros(v.shape[0], v.shape[1], q.shape[-1], v.shape[-1], device=q.device)
    out = []
    for n in range(qc.shape[2]):
        D = U[:, :, n] - torch.matmul(W[:, :, n], C)
        out.append(torch.matmul(qd[:, :, n], C) + torch.matmul(P[:, :, n], D))
        C = c_all[:, :, n] * C + torch.matmul(kd[:, :, n], D)
    return torch.cat(out, 2)[:, :, :S].to(v.dtype), C


# ------------------------------------------------------------------------------------- what a pass is
def work(case):
    esz = ESZ[case["dtype"]]
    if case["kind"] == "glu":
        T, D, F = case["T"], case["D"], case["F"]
        bytes_, flops = (T * D + 2 * F * D + T * F) * esz, 4 * T * D * F
        if case["train"]:
            bytes_, flops = bytes_ + (T * F + T * D + 2 * F * D) * esz, 3 * flops
        return {"bytes": bytes_, "flops": flops}
    B, NH, NHK, DQK, DV = (case[n] for n in ("B", "NH", "NHK", "DQK", "DV"))
    S = case.get("S", 1)
    # a token and head: C^T k, the update and C^T q; backward: three products with the state's gradient, three with the state
    rows, gates, states = B * S * (2 * NHK * DQK + NH * DV) * esz, 2 * B * NH * S * ESZ[case["gate"]], B * NH * DQK * DV * 4
    bytes_, flops = rows + B * S * NH * DV * esz + gates, 6 * B * NH * S * DQK * DV
    if case["kind"] != "chunk" or case["state"]:
        bytes_ += 2 * states
    if case.get("train"):
        bytes_, flops = bytes_ + rows + B * S * NH * DV * esz + gates + (2 * states if case["state"] else 0), 3 * flops
    return {"bytes": bytes_, "flops": flops}


# ------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    if case["kind"] == "glu":
        x, wg, wu, dh = (None if t is None else t.double() for t in _inputs(case, seed))
        a, u = x @ wg.mT, x @ wu.mT
        act = torch.nn.functional.silu(a)
        if not case["train"]:
            return act * u
        sig = torch.special.expit(a)
        da, du = dh * u * torch.lerp(sig, torch.ones_like(sig), act), dh * act
        return act * u, da @ wg + du @ wu, da.mT @ x, du.mT @ x
    given, dh, dc = _inputs(case, seed)
    q, k, v, g, beta, c0 = (None if t is None else t.double() for t in given)
    one = case["kind"] == "step"
    if one:
        q, k, v, g, beta = (t.unsqueeze(2) for t in (q, k, v, g, beta))
    B, NH, S, DV = v.shape
    DQK, scale, shared = q.shape[-1], q.shape[-1] ** -0.5, NH // q.shape[1]
    q, k = (t[:, :, None].expand(-1, -1, shared, -1, -1).reshape(B, NH, S, DQK) for t in (q, k))
    a = torch.exp(g)
    C = torch.zeros(B, NH, DQK, DV, dtype=torch.float64, device=DEV) if c0 is None else c0
    train = bool(case.get("train"))
    h, d, before = torch.empty_like(v), torch.empty_like(v), []
    for t in range(S):
        if train:
            before.append(C)
        kt = k[:, :, t]
        C = C * a[:, :, t, None, None]
        d[:, :, t] = v[:, :, t] - (kt.unsqueeze(-2) @ C).squeeze(-2)
        C = torch.addcmul(C, kt.unsqueeze(-1), (beta[:, :, t, None] * d[:, :, t]).unsqueeze(-2))
        h[:, :, t] = (q[:, :, t].unsqueeze(-2) @ C).squeeze(-2) * scale
    if one:
        return h[:, :, 0], C
    if not train:
        return (h, C) if case["kind"] == "short" or case["state"] else h
    # back through the recurrence, G the gradient of the state behind token t
    dh = dh.double() * scale
    G = torch.zeros_like(C) if dc is None else dc.double()
    last, after = C, C
    dq, dk, dv, dg, db = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(g), torch.empty_like(g)
    for t in reversed(range(S)):
        kt, dht, at, bt = k[:, :, t], dh[:, :, t], a[:, :, t], beta[:, :, t]
        dq[:, :, t] = (after @ dht.unsqueeze(-1)).squeeze(-1)
        G = torch.addcmul(G, q[:, :, t].unsqueeze(-1), dht.unsqueeze(-2))
        kG = (kt.unsqueeze(-2) @ G).squeeze(-2)
        db[:, :, t] = torch.linalg.vecdot(kG, d[:, :, t])
        e = bt[..., None] * kG
        dv[:, :, t] = e
        # the state as decayed: S = C + k (b d)^T, d = v - C^T k
        old = before.pop()
        decayed = old * at[..., None, None]
        dk[:, :, t] = (G @ (bt[..., None] * d[:, :, t]).unsqueeze(-1) - decayed @ e.unsqueeze(-1)).squeeze(-1)
        G = torch.addcmul(G, kt.unsqueeze(-1), e.unsqueeze(-2), value=-1.0)
        dg[:, :, t] = (G * decayed).sum((-2, -1))
        G = G * at[..., None, None]
        after = old
    dq, dk = (t.reshape(B, NH // shared, shared, S, DQK).sum(2) for t in (dq, dk))
    return (h, last, dq, dk, dv, dg, db, G) if case["state"] else (h, dq, dk, dv, dg, db)
