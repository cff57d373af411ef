"""The gated linear unit of a feed-forward block, with its gradients, on HIP (``csrc/gated_linear.hip``)."""

from __future__ import annotations

from torch import Tensor

from .ops import GLU_ACTS, gated_linear_op

__all__ = ["gated_linear_unit"]


def gated_linear_unit(x: Tensor, weight_gate: Tensor, weight_up: Tensor, activation: str = "silu") -> Tensor:
    """``act(x weight_gate^T) * (x weight_up^T)``: both projections of a SwiGLU (or, "gelu", GeGLU) block in one kernel.

    x [..., D], weights [F, D] (``nn.Linear``'s), bfloat16 or float16, one dtype; the result [..., F].  The products are
    float32 until the result's one rounding.  "gelu" is the exact one, by erf.  Up to 16 tokens (without a gradient) the
    weights are streamed past them.  Differentiable in x and both weights, once: the forward then keeps both products in
    float32.
    """
    if activation not in GLU_ACTS:
        raise ValueError(f"gated_linear_unit: activation must be one of {sorted(GLU_ACTS)}, got {activation!r}")
    return gated_linear_op(x, weight_gate, weight_up, GLU_ACTS[activation], False)[0]
