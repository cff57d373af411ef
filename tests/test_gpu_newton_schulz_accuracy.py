"""How far newton_schulz may be from the iteration in 64 bits, by bars that do not know how the kernels store a matrix.

f is the error of the same iteration with float32 products.  What rounding leaves in a direction of a small singular
value grows with it, 3.44-fold a step of Muon's coefficients, so an exactly low-rank matrix is the hard case.

* float16 and float32: 2 f, a rounding of the type, and 2^-21 a step (a pair of f16 holds 22 bits)."""

import pytest
import torch

from helpers import dev

pytestmark = pytest.mark.gpu

F32, F16 = torch.float32, torch.float16
MUON = (3.4445, -4.7750, 2.0315)
ROUNDING = {F16: 2.0 ** -11, F32: 2.0 ** -24}


def iterate(G, triples, eps=1e-7):
    tall = G.shape[0] > G.shape[1]
    X = G.mT if tall else G
    X = X / (torch.sqrt((X * X).sum()) + eps)
    for a, b, c in triples:
        A = torch.matmul(X, X.mT.contiguous())
        X = a * X + torch.matmul(b * A + c * torch.matmul(A, A), X)
    return X.mT if tall else X


def error(x, want):
    return float(torch.linalg.matrix_norm(x.double() - want) / torch.linalg.matrix_norm(want))


def matrix(kind, rank, m, n, dtype):
    """Exact in dtype for "exact" and the kinds of repeated rows; otherwise of that rank before it is rounded."""
    g = torch.Generator().manual_seed(rank + m)
    if kind == "spread":
        x = torch.randn(m, n, generator=g)
    elif kind == "low rank":
        x = torch.randn(m, rank, generator=g) @ torch.randn(rank, n, generator=g)
    elif kind == "exact":
        x = torch.randint(-2, 3, (m, rank), generator=g).float() @ torch.randint(-2, 3, (rank, n), generator=g).float()
    elif kind == "few rows":
        x = torch.zeros(m, n)
        x[torch.randperm(m, generator=g)[:rank]] = torch.randn(rank, n, generator=g)
    elif kind == "repeated rows":
        x = torch.randn(rank, n, generator=g)[torch.randint(rank, (m,), generator=g)]
    else:  # blocks of one value
        x = (torch.arange(m)[:, None] % rank == torch.arange(n) % rank).float()
    return x.to(dtype).to(dev())


KINDS = [("spread", 0), ("low rank", 8), ("low rank", 32), ("exact", 8), ("exact", 32), ("few rows", 4), ("repeated rows", 4),
         ("blocks", 3)]
# in one workgroup (the first, for pairs too), tiles, few rows with a long sum, tall
SHAPES = [(64, 100), (128, 256), (129, 129), (64, 1024), (700, 300), (64, 2300)]


@pytest.mark.parametrize("kind,rank", KINDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("steps", [6, 10])
def test_many_steps(gpu_case, kind, rank, shape, dtype, steps):
    import xlstm_hip
    G, triples = matrix(kind, rank, *shape, dtype), (MUON,) * steps
    want = iterate(G.double(), triples)
    bar = 2 * error(iterate(G.float(), triples), want) + ROUNDING[dtype] + steps * 2.0 ** -21
    off = error(xlstm_hip.newton_schulz(G, steps), want)
    assert off <= bar, f"{off:.2e} over {bar:.2e}"
