"""How far newton_schulz may be from the iteration in 64 bits, by bars that do not know how the kernels store a matrix.

f is the error of the same iteration with float32 products, u = 2^-8 the largest relative error of one rounding to
bfloat16.  What rounding leaves in a direction of a small singular value grows with it, 3.44-fold a step of Muon's
coefficients, so an exactly low-rank matrix is the hard case.

* float16 and float32: 2 f, a rounding of the type, and 2^-21 a step (a pair of f16 holds 22 bits).
* bfloat16 where products of single f16 planes would be off by more than the result's rounding (more than five of
  Muon's steps, sixteen cubic ones): the same with u, as if the products were float32's.
* bfloat16, five of Muon's steps or fewer: 2 u for a matrix of unequal values, 4 u where rows repeat, whose roundings
  are equal and add up.  A step stores A, P and X to 2^-11 at worst; with |P| up to 2.7 and X in P X and twice in A, that
  is 7.6 * 2^-11 = 3.7e-3 if all three roundings lie the same way, 2e-4 * 4.2 = 0.9e-3 (a fifth of u) as they fall; the
  steps behind it multiply it by up to 1.6 for the large singular values: 5.2 such steps at most, 1.1 u."""

import pytest
import torch

from helpers import dev

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
MUON = (3.4445, -4.7750, 2.0315)
U = 2.0 ** -8
ROUNDING = {BF16: U, F16: 2.0 ** -11, F32: 2.0 ** -24}


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
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("steps", [6, 10])
def test_many_steps(gpu_case, kind, rank, shape, dtype, steps):
    import xlstm_hip
    G, triples = matrix(kind, rank, *shape, dtype), (MUON,) * steps
    want = iterate(G.double(), triples)
    bar = 2 * error(iterate(G.float(), triples), want) + ROUNDING[dtype] + steps * 2.0 ** -21
    off = error(xlstm_hip.newton_schulz(G, steps), want)
    assert off <= bar, f"{off:.2e} over {bar:.2e}"


@pytest.mark.parametrize("kind,rank", KINDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("steps", [1, 3, 5])
def test_bfloat16_few_steps(gpu_case, kind, rank, shape, steps):
    import xlstm_hip
    G, triples = matrix(kind, rank, *shape, BF16), (MUON,) * steps
    want = iterate(G.double(), triples)
    off = error(xlstm_hip.newton_schulz(G, steps), want)
    assert off <= (4 if kind in ("repeated rows", "blocks") else 2) * U, f"{off:.2e}"


@pytest.mark.parametrize("kind,rank", KINDS)
@pytest.mark.parametrize("shape", SHAPES[:4], ids=str)
def test_cubic_steps(gpu_case, kind, rank, shape):
    """Sixteen steps of the cubic iteration, which takes small singular values 1.5-fold a step."""
    import xlstm_hip
    G, triples = matrix(kind, rank, *shape, BF16), ((1.5, -0.5, 0.0),) * 16
    want = iterate(G.double(), triples)
    bar = 2 * error(iterate(G.float(), triples), want) + U + 16 * 2.0 ** -21
    off = error(xlstm_hip.newton_schulz(G, 16, triples), want)
    assert off <= bar, f"{off:.2e} over {bar:.2e}"


def test_batch_stream_and_graph_of_many_steps(gpu_case):
    """bfloat16 matrices by pairs: a matrix of a batch has the bits it has alone, on another stream and in a replay too."""
    import xlstm_hip
    G = torch.stack([matrix("low rank", 8, 150, 210, BF16), matrix("spread", 0, 150, 210, BF16), matrix("exact", 8, 150, 210, BF16)])
    alone = torch.stack([xlstm_hip.newton_schulz(x, 8) for x in G])
    assert torch.equal(xlstm_hip.newton_schulz(G, 8), alone)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = xlstm_hip.newton_schulz(G * 1.0, 8)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, alone)
    held_in = G.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = xlstm_hip.newton_schulz(held_in, 8)
    for k in range(4):
        held_in.copy_(G.roll(k, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, alone.roll(k, 0)), f"replay {k}"


@pytest.mark.parametrize("eps", [1e-7, 1e-20, 1e-30])
@pytest.mark.parametrize("shape", [(40, 60), (3, 130, 257)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_zero_matrix(gpu_case, eps, shape, dtype):
    """0 / (0 + eps) is 0 for every eps above 0."""
    import xlstm_hip
    assert not xlstm_hip.newton_schulz(torch.zeros(shape, dtype=dtype, device=dev()), eps=eps).any()
    if len(shape) == 3:
        G = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev())
        G[1] = 0
        got = xlstm_hip.newton_schulz(G, eps=eps)
        assert not got[1].any() and bool(got[[0, 2]].isfinite().all()) and bool(got[[0, 2]].any())


# of eps: far below, where five of Muon's steps (485-fold) just reach 1, and up to it
@pytest.mark.parametrize("ratio", [1e-30, 1e-12, 1e-6, 1 / 485, 1e-2, 0.03, 0.1, 1.0])
@pytest.mark.parametrize("shape", [(70, 150), (100, 120), (1024, 2048)], ids=str)
@pytest.mark.parametrize("coefficients", [MUON, (1.0, 0.8, 0.0)], ids=["Muon", "growing with the value"])
def test_norm_below_eps(gpu_case, ratio, shape, coefficients):
    import xlstm_hip
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(4))
    G, steps = (x / x.norm() * (ratio * 1e-3)).to(dev()), 5 if coefficients is MUON else 2
    triples = (coefficients,) * steps
    want = iterate(G.double(), triples, 1e-3)
    bar = 2 * error(iterate(G, triples, 1e-3), want) + 2.0 ** -24 + steps * 2.0 ** -21
    off = error(xlstm_hip.newton_schulz(G, steps, coefficients, eps=1e-3), want)
    assert off <= bar, f"{off:.2e} over {bar:.2e}"
