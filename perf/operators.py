"""Performance cases of the training operators around the mLSTM kernels: layer norm (over the last axis, and over
each head's values) with its backward pass, and the orthogonalisation of a weight's update by Newton-Schulz products.

A case is a dict of plain values; ``kind`` names the call:

* ``norm``   ``layer_norm`` of ``rows`` rows of ``D`` values
* ``heads``  ``multi_head_layer_norm`` of the chunkwise kernels' output [B, NH, S, DH], written [B, S, NH * DH]
* ``ortho``  ``newton_schulz`` of ``batch`` matrices [m, n], five steps

``train`` adds the backward pass (gradients of input, weight and bias); ``param`` is the type of weight and bias.
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
EPS = 1e-5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
NORM_EPS = 1e-7

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
        # serving: one token for each of 8 sequences at d 4096 (latency)
        dict(name="norm_token", kind="norm", rows=8, D=4096, dtype="bf16", param="bf16", train=False),
        # a batch of prompts, 8192 tokens at d 4096 (a stream through memory)
        dict(name="norm_prompt", kind="norm", rows=8192, D=4096, dtype="bf16", param="bf16", train=False),
        # training at d 4096: 8192 tokens, float32 weights beside bf16 activations
        dict(name="norm_train", kind="norm", rows=8192, D=4096, dtype="bf16", param="f32", train=True),
        # float32 training of the smaller model, d 2048, a ragged number of tokens
        dict(name="norm_train_f32", kind="norm", rows=2011, D=2048, dtype="f32", param="f32", train=True),
        # rows of an odd length, which no 16-byte vector fits
        dict(name="norm_train_odd", kind="norm", rows=4001, D=1333, dtype="f16", param="f16", train=True),
        # the sLSTM layer's heads over one prompt
        dict(name="heads_prompt", kind="heads", B=1, NH=4, S=777, DH=512, dtype="bf16", param="bf16", train=False),
        # training behind the chunkwise kernel at the 7B head shape
        dict(name="heads_train", kind="heads", B=2, NH=8, S=4096, DH=512, dtype="bf16", param="bf16", train=True),
        # a small projection on its own (latency: fifteen dependent products)
        dict(name="ortho_small", kind="ortho", batch=1, m=128, n=128, dtype="bf16"),
        # the q / k projections of the smaller model's blocks, together
        dict(name="ortho_batch", kind="ortho", batch=12, m=1024, n=2048, dtype="bf16"),
        # a float32 update of odd sizes
        dict(name="ortho_f32", kind="ortho", batch=1, m=1777, n=1000, dtype="f32"),
        # the 7B model's square output projection
        dict(name="ortho_square", kind="ortho", batch=1, m=4096, n=4096, dtype="bf16"),
        # the 7B model's feed-forward weight: the largest matrix that training updates
        dict(name="ortho_ffn", kind="ortho", batch=1, m=10944, n=4096, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "heads", "ortho", "ortho"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    param = rng.choice((dtype, "f32"))
    train = rng.random() < 0.6
    if kind == "norm":
        D = _log(rng, 64, 16384)
        D = rng.choice((D, (D + 7) // 8 * 8))
        return dict(kind=kind, rows=_log(rng, 1, (1 << 25) // D), D=D, dtype=dtype, param=param, train=train)
    if kind == "heads":
        B, NH, DH = rng.choice((1, 2, 3, 8)), rng.choice((2, 4, 8)), rng.choice((64, 96, 128, 200, 256, 320, 512))
        return dict(kind=kind, B=B, NH=NH, S=_log(rng, 1, 8192 // B), DH=DH, dtype=dtype, param=param, train=train)
    while True:
        case = dict(kind=kind, batch=rng.choice((1, 1, 2, 4, 12)), m=_log(rng, 32, 10944), n=_log(rng, 32, 10944), dtype=dtype)
        w = work(case)
        if w["flops"] * (3 if dtype == "f32" else 1) <= 4e12 and w["bytes"] <= 2e8:
            return case


# ------------------------------------------------------------------------------------- inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DT[case["dtype"]]
    if case["kind"] == "ortho":
        # a gradient's spectrum: most of its weight in some directions, the rest spread over all
        b, m, n = case["batch"], case["m"], case["n"]
        r = max(1, min(m, n) // 16)
        strong = torch.matmul(_randn(g, b, m, r), _randn(g, b, r, n)) / math.sqrt(r)
        return (((strong + 0.3 * _randn(g, b, m, n)) * 1e-3).to(dt),)
    if case["kind"] == "norm":
        C, lead, groups = case["D"], (case["rows"],), case["D"]
        shape = lead + (C,)
    else:
        C, shape = case["NH"] * case["DH"], (case["B"], case["NH"], case["S"], case["DH"])
        groups = case["DH"]
    # activations with a mean and a scale of each channel, as a residual stream has
    x = _randn(g, *shape) * (0.5 + torch.rand(groups, generator=g, device=DEV)) + 0.3 * _randn(g, groups)
    w, b = 1.0 + 0.1 * _randn(g, C), 0.1 * _randn(g, C)
    out = (case["rows"], C) if case["kind"] == "norm" else (case["B"], case["S"], C)
    dy = 0.1 * _randn(g, *out) if case["train"] else None
    pt = DT[case["param"]]
    return x.to(dt), w.to(pt), b.to(pt), None if dy is None else dy.to(dt)


def prepare(case, seed):
    state = dict(case=case, inputs=_inputs(case, seed))
    if case.get("train"):
        for t in state["inputs"][:3]:
            t.requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------- one pass
def run(state):
    case, inputs = state["case"], state["inputs"]
    if case["kind"] == "ortho":
        return _framework().newton_schulz(inputs[0]) if own else _plain_ortho(inputs[0])
    if not own:
        with torch.no_grad():
            return _plain_norm(case, *inputs)
    hip = _framework()
    x, w, b, dy = inputs
    y = hip.layer_norm(x, w, b, EPS) if case["kind"] == "norm" else hip.multi_head_layer_norm(x, w, b, EPS)
    if not case["train"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))


def _plain_norm(case, x, w, b, dy):
    """Layer norm and its gradients from the formula, in 32 bits:
    h = (x - mean) / sqrt(var + eps), y = h w + b; with g = dy w:
    dx = (g - mean(g) - h mean(g h)) / sqrt(var + eps), dw = sum dy h, db = sum dy."""
    heads = case["kind"] == "heads"
    split = (case["NH"], case["DH"]) if heads else (case["D"],)
    xf = x.float()
    if heads:
        xf = xf.transpose(1, 2)
    wf, bf = w.float().view(split), b.float().view(split)
    centred = xf - xf.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    h = centred * rstd
    y = (h * wf + bf).to(x.dtype)
    if heads:
        y = y.reshape(y.shape[0], y.shape[1], -1)
    if not case["train"]:
        return y
    d = dy.float().view(xf.shape)
    g = d * wf
    dx = ((g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True)) * rstd).to(x.dtype)
    lead = tuple(range(xf.dim() - len(split)))
    dw, db = (d * h).sum(lead).view(-1).to(w.dtype), d.sum(lead).view(-1).to(b.dtype)
    return y, dx.transpose(1, 2) if heads else dx, dw, db


def _plain_ortho(x):
    """X = G / (|G| + eps); five times X = a X + (b X X^T + c (X X^T)^2) X, on the side with fewer rows, in 32 bits."""
    a, b, c = COEFFICIENTS
    X = x.float()
    if x.shape[-2] > x.shape[-1]:
        X = X.transpose(-2, -1)
    X = X / (torch.sqrt((X * X).sum((-2, -1), keepdim=True)) + NORM_EPS)
    for _ in range(STEPS):
        A = torch.matmul(X, X.transpose(-2, -1))
        X = a * X + torch.matmul(b * A + c * torch.matmul(A, A), X)
    if x.shape[-2] > x.shape[-1]:
        X = X.transpose(-2, -1)
    return X.to(x.dtype)


# ------------------------------------------------------------------------------------- what a pass is
def work(case):
    esz = ESZ[case["dtype"]]
    if case["kind"] == "ortho":
        # X X^T and its square are symmetric: half of each product
        M, N, B = min(case["m"], case["n"]), max(case["m"], case["n"]), case["batch"]
        return {"bytes": 2 * B * M * N * esz, "flops": STEPS * B * (M * M * N + M ** 3 + 2 * M * M * N)}
    if case["kind"] == "norm":
        count, C = case["rows"] * case["D"], case["D"]
    else:
        count, C = case["B"] * case["S"] * case["NH"] * case["DH"], case["NH"] * case["DH"]
    psz = ESZ[case["param"]]
    bytes_ = 2 * count * esz + 2 * C * psz
    flops = 8 * count
    if case["train"]:
        bytes_ += 2 * count * esz + 2 * C * psz  # dy in, dx out (x is the forward's), dw and db out
        flops += 14 * count
    return {"bytes": bytes_, "flops": flops}


# ------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    inputs = _inputs(case, seed)
    if case["kind"] == "ortho":
        # the steps' factors are polynomials of G G^T: their product Q is formed beside it, then X = Q G / (|G| + eps)
        G = inputs[0].double()
        tall = G.shape[-2] > G.shape[-1]
        G = G.mT if tall else G
        G = G / (torch.linalg.matrix_norm(G)[:, None, None] + NORM_EPS)
        a, b, c = COEFFICIENTS
        eye = torch.eye(G.shape[-2], dtype=torch.float64, device=G.device)
        A, Q = G @ G.mT, eye
        for _ in range(STEPS):
            F = a * eye + b * A + c * (A @ A)
            Q, A = F @ Q, F @ A @ F
        X = Q @ G
        return X.mT if tall else X
    x, w, b, dy = (None if t is None else t.double() for t in inputs)
    heads = case["kind"] == "heads"
    C = w.numel()
    if heads:
        NH, DH = case["NH"], case["DH"]
        rows = x.permute(0, 2, 1, 3).reshape(-1, NH, DH)
    else:
        rows = x.reshape(-1, 1, C)
    var, mean = torch.var_mean(rows, dim=-1, correction=0, keepdim=True)
    rstd = torch.rsqrt(var + EPS)
    h = ((rows - mean) * rstd).reshape(-1, C)
    shape = (case["B"], case["S"], C) if heads else (case["rows"], C)
    y = torch.addcmul(b, h, w).reshape(shape)
    if not case["train"]:
        return y
    d = dy.reshape(-1, C)
    n = rows.shape[-1]
    g = (d * w).reshape(rows.shape)
    hh = h.reshape(rows.shape)
    # the projection of g off the constant and off h, within each normalised group
    dx = rstd / n * (n * g - g.sum(-1, keepdim=True) - hh * torch.linalg.vecdot(g, hh)[..., None])
    if heads:
        dx = dx.reshape(case["B"], case["S"], NH, DH).permute(0, 2, 1, 3)
    return y, dx.reshape(x.shape) if not heads else dx, torch.linalg.vecdot(d, h, dim=0), d.sum(0)
