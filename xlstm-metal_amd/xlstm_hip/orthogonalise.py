"""Orthogonalised updates, on HIP (``csrc/newton_schulz.hip``).

``newton_schulz`` brings the singular values of a matrix (a gradient, its momentum) to about 1 and leaves the singular
vectors alone, by products alone: what the Muon optimiser applies to a weight in place of the gradient.
"""

from __future__ import annotations

from typing import Sequence, Union

from torch import Tensor

from .ops import newton_schulz_op

__all__ = ["newton_schulz", "MUON_COEFFICIENTS"]

#: Muon's quintic: steep at 0 (small singular values grow 3.4-fold a step), settling in [0.7, 1.2].
MUON_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def newton_schulz(x: Tensor, steps: int = 5, coefficients: Sequence[Union[float, Sequence[float]]] = MUON_COEFFICIENTS,
                  eps: float = 1e-7) -> Tensor:
    """X = x / (|x|_F + eps), then ``steps`` times X = a X + (b X X^T + c (X X^T)^2) X, for each matrix [..., m, n].

    ``coefficients`` is (a, b, c), or one such triple for each step.  The result has x's dtype.  float16 and float32 run
    products of f16 pairs, as exact as float32 products; bfloat16 runs plain f16 products, at about a third of their time,
    for up to five of Muon's steps: 1.7e-3 to 2.1e-3 of the norm off for spread singular values (the rounding to bfloat16
    alone: 1.65e-3), up to 5.3e-3 for matrices of low rank and 1e-2 where rows repeat.  More such steps, which would let that
    grow, run pairs.  Cast a float32 momentum to bfloat16 first, as Muon does, where that much is enough.  Coefficients
    that take the singular values past 8 raise ``ValueError``.  Not differentiable.
    """
    if steps < 1:
        raise ValueError(f"newton_schulz: steps must be at least 1, got {steps}")
    triples = [coefficients] * steps if not hasattr(coefficients[0], "__len__") else list(coefficients)
    if len(triples) != steps or any(len(t) != 3 for t in triples):
        raise ValueError(f"newton_schulz: coefficients must be (a, b, c) or {steps} such triples, got {coefficients}")
    return newton_schulz_op(x, [float(c) for t in triples for c in t], float(eps))
