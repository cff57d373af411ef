"""Trains a small mLSTM language model with this library's operators:

    python examples/train_block.py --steps 60

Each block is x + mLSTM(LayerNorm(x)), then x + FFN(LayerNorm(x)): the norms are ``layer_norm``, the sequence mixing
``mlstm_chunkwise`` with its backward kernels, the heads' norm behind it ``multi_head_layer_norm`` on the chunkwise
output as it lies.  The blocks' matrices are updated by Muon (momentum, orthogonalised by ``newton_schulz``, matrices of
one shape together), everything else by AdamW.  The data are sequences that count up by a step of their own (1 to 4)
from a random token: the last token alone leaves a loss of log 4, the steps before it tell the next token.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xlstm-metal_amd"))
import xlstm_hip  # noqa: E402


class LayerNorm(nn.Module):
    """float32 weights beside activations of any type."""

    def __init__(self, d: int) -> None:
        super().__init__()
        self.weight, self.bias = nn.Parameter(torch.ones(d)), nn.Parameter(torch.zeros(d))

    def forward(self, x):
        return xlstm_hip.layer_norm(x, self.weight, self.bias)


class Block(nn.Module):
    def __init__(self, d: int, heads: int) -> None:
        super().__init__()
        self.heads = heads
        self.norm1, self.norm2 = LayerNorm(d), LayerNorm(d)
        self.q, self.k = nn.Linear(d, d // 2, bias=False), nn.Linear(d, d // 2, bias=False)
        self.v, self.o, self.out = (nn.Linear(d, d, bias=False) for _ in range(3))
        self.gates = nn.Linear(d, 2 * heads)
        self.head_weight = nn.Parameter(torch.ones(d))
        self.up, self.down = nn.Linear(d, 2 * d, bias=False), nn.Linear(2 * d, d, bias=False)
        with torch.no_grad():  # forget gates near 1
            self.gates.bias.copy_(torch.cat([torch.zeros(heads), torch.full((heads,), 3.0)]))

    def matrices(self):
        return [m.weight for m in (self.q, self.k, self.v, self.o, self.out, self.up, self.down)]

    def forward(self, x):
        B, S, _ = x.shape
        y = self.norm1(x)
        w = lambda m: F.linear(y, m.weight.to(y.dtype))  # noqa: E731  (float32 weights, products in x's type)
        q, k, v = (w(m).view(B, S, self.heads, -1).transpose(1, 2) for m in (self.q, self.k, self.v))
        i, f = F.linear(y.float(), self.gates.weight, self.gates.bias).transpose(1, 2).contiguous().chunk(2, dim=1)
        h = xlstm_hip.mlstm_chunkwise(q.contiguous(), k.contiguous(), v.contiguous(), i.contiguous(), f.contiguous(),
                                      chunk_size=64)
        h = xlstm_hip.multi_head_layer_norm(h, self.head_weight)
        x = x + F.linear(h * torch.sigmoid(w(self.o)), self.out.weight.to(x.dtype))
        y = self.norm2(x)
        return x + F.linear(F.silu(F.linear(y, self.up.weight.to(y.dtype))), self.down.weight.to(y.dtype))


class Model(nn.Module):
    def __init__(self, vocab: int, d: int, blocks: int, heads: int, dtype: torch.dtype) -> None:
        super().__init__()
        self.dtype = dtype
        self.embedding = nn.Embedding(vocab, d)
        self.blocks = nn.ModuleList(Block(d, heads) for _ in range(blocks))
        self.norm, self.head = LayerNorm(d), nn.Linear(d, vocab, bias=False)

    def forward(self, tokens):
        x = self.embedding(tokens).to(self.dtype)
        for block in self.blocks:
            x = block(x)
        return F.linear(self.norm(x).float(), self.head.weight)


class Muon(torch.optim.Optimizer):
    """W -= lr sqrt(max(1, rows / columns)) newton_schulz(momentum), matrices of one shape in one call."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95) -> None:
        super().__init__(params, dict(lr=lr, momentum=momentum))

    @torch.no_grad()
    def step(self):
        for group in self.param_groups:
            shapes = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    state["momentum"] = torch.zeros_like(p)
                state["momentum"].lerp_(p.grad, 1 - group["momentum"])
                shapes.setdefault(p.shape, []).append((p, p.grad.lerp(state["momentum"], group["momentum"])))
            for (rows, cols), pairs in shapes.items():
                updates = xlstm_hip.newton_schulz(torch.stack([u for _, u in pairs]).to(torch.bfloat16))
                for (p, _), update in zip(pairs, updates):
                    p.add_(update.to(p.dtype), alpha=-group["lr"] * max(1.0, rows / cols) ** 0.5)


def batch_of(g: torch.Generator, batch: int, length: int, vocab: int, device):
    first, stride = torch.randint(vocab, (batch, 1), generator=g), torch.randint(1, 5, (batch, 1), generator=g)
    return ((first + stride * torch.arange(length + 1)) % vocab).to(device)


def train(steps: int = 60, d: int = 256, blocks: int = 2, heads: int = 4, batch: int = 8, length: int = 256, vocab: int = 64,
          device: str = "cuda:0", seed: int = 0, report=print):
    """The loss of every step."""
    torch.manual_seed(seed)
    model = Model(vocab, d, blocks, heads, torch.bfloat16).to(device)
    matrices = [w for b in model.blocks for w in b.matrices()]
    held = {id(w) for w in matrices}
    optimisers = [Muon(matrices), torch.optim.AdamW([p for p in model.parameters() if id(p) not in held], lr=3e-3)]
    g = torch.Generator().manual_seed(seed)
    losses = []
    for step in range(steps):
        tokens = batch_of(g, batch, length, vocab, device)
        loss = F.cross_entropy(model(tokens[:, :-1]).flatten(0, 1), tokens[:, 1:].flatten())
        for o in optimisers:
            o.zero_grad(set_to_none=True)
        loss.backward()
        for o in optimisers:
            o.step()
        losses.append(float(loss.detach()))
        if step % 10 == 0 or step + 1 == steps:
            report(f"step {step:4d}  loss {losses[-1]:.4f}")
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--d-model", type=int, default=256)
    ap.add_argument("--blocks", type=int, default=2)
    a = ap.parse_args()
    train(a.steps, a.d_model, a.blocks)
