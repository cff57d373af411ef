"""Newton-Schulz orthogonalisation on the GPU against the iteration in 64 bits.

The bar of a case is twice what its arithmetic must lose, as relative error in the Frobenius norm: the iteration in
64 bits with every stored matrix rounded as the kernels store it (f16 at a power-of-two scale, or hi + lo pairs), plus
the iteration in float32 where float32 sums matter (f16 and float32 inputs), plus the result's own rounding (its type's
half unit in the last place).  Single values: 40 times that, of the root mean square of all values plus their own."""

import pytest
import torch

from helpers import dev

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
MUON = (3.4445, -4.7750, 2.0315)
HALF_ULP = {BF16: 2.0 ** -9, F16: 2.0 ** -12, F32: 2.0 ** -25}


def iterate(G, triples, eps=1e-7):
    """The definition, in G's own type."""
    tall = G.shape[-2] > G.shape[-1]
    X = G.mT if tall else G
    X = X / (torch.sqrt((X * X).sum((-2, -1), keepdim=True)) + eps)
    for a, b, c in triples:
        A = torch.matmul(X, X.mT.contiguous())
        X = a * X + torch.matmul(b * A + c * torch.matmul(A, A), X)
    return X.mT if tall else X


def rounded(G, triples, pairs):
    """The iteration in 64 bits with the kernels' stored matrices: X, A and P in f16 (X and the linear term of the middle
    steps as a pair, P's diagonal apart; with `pairs` all of them as pairs)."""
    def store(x, scale):
        hi = (x * scale).to(F16).double()
        return hi / scale, (x * scale - hi).to(F16).double() / scale

    def product(p, q):
        return p[0] @ q[0].mT + (p[0] @ q[1].mT + p[1] @ q[0].mT if pairs else 0.0)

    X = G.double()
    X = X.mT if X.shape[-2] > X.shape[-1] else X
    norm = torch.linalg.matrix_norm(X)[..., None, None] + 1e-7
    start = 2.0 ** (13 - torch.ceil(torch.log2(norm)))
    S = tuple(t / (start * norm) for t in store(X * start, 1.0))
    for k, (a, b, c) in enumerate(triples):
        A = store(product(S, S), 256.0)
        full = A[0] + (A[1] if pairs else 0.0)
        P = b * full + c * product(A, A)
        D = torch.zeros_like(P[..., :1]) if pairs else torch.diagonal(P, dim1=-2, dim2=-1).unsqueeze(-1)
        P = store(P - torch.diag_embed(D.squeeze(-1)), 64.0)
        linear = S[0] + (S[1] if pairs or 1 <= k <= len(triples) - 2 else 0.0)
        X = (a + D) * linear + product(P, tuple(t.mT for t in S))
        S = store(X, 256.0)
    return X.mT if G.shape[-2] > G.shape[-1] else X


def error(x, want):
    return torch.linalg.matrix_norm(x.double() - want) / torch.linalg.matrix_norm(want).clamp_min(1e-300)


def check(got, G, triples=(MUON,) * 5, eps=1e-7):
    want = iterate(G.double(), triples, eps)
    bar = error(rounded(G, triples, G.dtype != BF16), want) + HALF_ULP[G.dtype]
    if G.dtype != BF16:
        bar = bar + error(iterate(G.float(), triples, eps), want)
    off = error(got, want)
    assert got.dtype == G.dtype and got.shape == G.shape
    assert bool((off <= 2 * bar).all()), f"off by {float((off / bar).max()):.2f} of the bar ({float(off.max()):.2e})"
    rms = torch.linalg.matrix_norm(want) / (G.shape[-2] * G.shape[-1]) ** 0.5
    single = (got.double() - want).abs() / (rms[..., None, None] + want.abs()).clamp_min(1e-300)
    assert bool((single.amax((-2, -1)) <= 40 * bar).all()), f"a value off by {float((single.amax((-2, -1)) / bar).max()):.1f}"


def gradient(shape, dtype, seed=0, kind="spread"):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    m, n = shape[-2:]
    k = max(1, min(m, n) // 16)
    x = 1e-3 * (r(*shape[:-1], k) @ r(*shape[:-2], k, n) / k ** 0.5 + 0.3 * r(*shape)) if kind == "spread" else 1e-3 * r(*shape)
    return x.to(dtype).to(dev())


# one value; vectors; less than a tile, a tile, just past it; odd; the largest in one workgroup and just past them; wide and tall; a long sum for few rows; batches
SHAPES = [(1, 1), (1, 9), (200, 1), (3, 5), (33, 17), (64, 64), (128, 128), (127, 129), (129, 128), (130, 257), (200, 333),
          (31, 2050), (2050, 31), (100, 5000), (513, 700), (1000, 777), (64, 256), (65, 200), (128, 256), (257, 128), (60, 257), (128, 130), (256, 64), (3, 65, 130), (2, 2, 140, 96), (17, 64, 64), (0, 8, 8),
          (8, 0)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_sizes(gpu_case, shape, dtype):
    import xlstm_hip
    G = gradient(shape, dtype, seed=sum(shape)) if 0 not in shape else torch.empty(shape, dtype=dtype, device=dev())
    got = xlstm_hip.newton_schulz(G)
    if 0 in shape:
        assert got.shape == G.shape
    else:
        check(got, G)


# every size of tile and depth of stages
@pytest.mark.parametrize("shape", [(1536, 1100), (2048, 2304), (2, 1300, 2600), (640, 6000), (4100, 2900), (6, 1000, 2000)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large(gpu_case, shape, dtype):
    import xlstm_hip
    G = gradient(shape, dtype, seed=3)
    check(xlstm_hip.newton_schulz(G), G)


@pytest.mark.parametrize("kind", ["gauss", "rank one", "orthogonal", "one value", "one row", "power", "outlier"])
@pytest.mark.parametrize("shape", [(96, 160), (260, 150)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_spectra(gpu_case, kind, shape, dtype):
    import xlstm_hip
    x = gradient(shape, F32, seed=5, kind="gauss")
    if kind == "rank one":
        x = x[:, :1] * x[:1] * 1e3
    elif kind in ("orthogonal", "power"):
        u, s, v = torch.linalg.svd(x.cpu(), full_matrices=False)
        s = torch.ones_like(s) if kind == "orthogonal" else torch.arange(1, len(s) + 1).float() ** -1.0
        x = (u * s @ v).to(dev())
    elif kind == "one value":
        x = torch.zeros_like(x)
        x[7, 11] = 3.0
    elif kind == "one row":
        x[1:] = 0
    elif kind == "outlier":
        x[5, 5] = 50.0
    G = x.to(dtype)
    check(xlstm_hip.newton_schulz(G), G)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e-8, 1.0, 1e18, 1e30])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scales(gpu_case, scale, dtype):
    """Far below eps the result is small, far above it does not overflow (nor does the square of a value)."""
    import xlstm_hip
    G = (gradient((70, 150), F32, seed=6) * 1e3 * scale).to(dtype)
    want = iterate(G.double(), (MUON,) * 5)
    got = xlstm_hip.newton_schulz(G)
    assert float(error(got, want)) <= (6e-3 if dtype == BF16 else 2e-5)


def test_zeros_and_special_values(gpu_case):
    """A zero matrix gives zeros; a NaN or an infinity stays in its matrix."""
    import xlstm_hip
    G = gradient((4, 90, 140), BF16, seed=7)
    alone = xlstm_hip.newton_schulz(G)
    G[1] = 0
    G[2, 3, 4], G[3, 5, 6] = float("nan"), float("inf")
    got = xlstm_hip.newton_schulz(G)
    assert torch.equal(got[0], alone[0]) and not got[1].any()
    assert bool(got[2].isnan().any()) and bool(got[3].isnan().any())


@pytest.mark.parametrize("triples", [[(1.5, -0.5, 0.0)], [(1.5, -0.5, 0.0)] * 12, [(2.0, -1.5, 0.5)] * 3,
                                     [(8.0, -22.0, 16.0), (2.2, -0.9, 0.12), (1.875, -1.25, 0.375), (1.875, -1.25, 0.375)]], ids=len)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_coefficients(gpu_case, triples, dtype):
    import xlstm_hip
    G = gradient((150, 220), dtype, seed=8)
    check(xlstm_hip.newton_schulz(G, len(triples), triples), G, triples)


@pytest.mark.parametrize("kind", ["transposed", "columns", "rows", "batch apart", "odd start"])
def test_strides(gpu_case, kind):
    import xlstm_hip
    base = gradient((3, 140, 301), BF16, seed=9)
    G = {"transposed": lambda: base.mT, "columns": lambda: base[:, :, 5:201], "rows": lambda: base[:, ::2],
         "batch apart": lambda: base[::2], "odd start": lambda: base.view(-1)[1:90 * 100 + 1].view(90, 100)}[kind]()
    got = xlstm_hip.newton_schulz(G)
    assert got.is_contiguous() and torch.equal(got, xlstm_hip.newton_schulz(G.clone(memory_format=torch.contiguous_format)))
    check(got, G)


def test_turned_alike(gpu_case):
    """The transpose of the result is the result of the transpose: the same products."""
    import xlstm_hip
    G = gradient((150, 400), F32, seed=10)
    assert torch.equal(xlstm_hip.newton_schulz(G.mT).mT, xlstm_hip.newton_schulz(G))


@pytest.mark.parametrize("shape", [(1, 100, 120), (5, 600, 400)], ids=str)
def test_other_stream_same_bits_and_graph(gpu_case, shape):
    import xlstm_hip
    G = gradient(shape, BF16, seed=11)
    first = xlstm_hip.newton_schulz(G)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = xlstm_hip.newton_schulz(G * 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, again)
    held_in = G.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = xlstm_hip.newton_schulz(held_in)
    for k in range(4):
        held_in.copy_(G.roll(k, -1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, xlstm_hip.newton_schulz(G.roll(k, -1))), f"replay {k}"


def test_refusals(gpu_case):
    import xlstm_hip
    G = gradient((8, 8), BF16)
    with pytest.raises(ValueError, match="matrix"):
        xlstm_hip.newton_schulz(G[0])
    with pytest.raises(ValueError, match="dtype"):
        xlstm_hip.newton_schulz(G.double())
    with pytest.raises(ValueError, match="out of range"):
        xlstm_hip.newton_schulz(G, 5, (8.0, 3.0, 2.0))
    with pytest.raises(ValueError, match="out of range"):
        xlstm_hip.newton_schulz(G, 1, (float("nan"), 0.0, 0.0))
    with pytest.raises(ValueError, match="eps"):
        xlstm_hip.newton_schulz(G, eps=-1.0)
    with pytest.raises(NotImplementedError, match="65536"):
        xlstm_hip.newton_schulz(torch.empty(1, 70000, dtype=BF16, device=dev()))
    x = G.clone().requires_grad_(True)
    with pytest.raises(RuntimeError):
        xlstm_hip.newton_schulz(x).float().sum().backward()
