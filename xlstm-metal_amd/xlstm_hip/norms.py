"""Layer norm with its gradients, on HIP (``csrc/layer_norm.hip``).

``layer_norm`` is ``torch.nn.functional.layer_norm`` over the last axis; ``multi_head_layer_norm`` norms each head of
the chunkwise kernels' output (``MultiHeadLayerNorm``, ``xlstm_metal/torch_native/blocks/mlstm/multihead_norm/
multihead_norm.py:5-40``) and reads it where it lies.  Statistics, sums and the weight's gradient are float32, every
output is rounded once; weight and bias have x's dtype or float32, and their gradients theirs.
"""

from __future__ import annotations

from typing import Optional

from torch import Tensor

from .ops import layer_norm_op

__all__ = ["layer_norm", "multi_head_layer_norm"]


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis of x; weight, bias [D] or None.

    Any strides with a contiguous last axis are read in place where the leading axes fold into two; the result is
    contiguous.  Differentiable in x, weight and bias.
    """
    return layer_norm_op(x, weight, bias, eps, 0)[0]


def multi_head_layer_norm(h: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-6,
                          heads_first: bool = True) -> Tensor:
    """Layer norm of every head over DH, as [B, S, NH * DH].

    h is [B, NH, S, DH] (``heads_first``, the chunkwise output) or [B, S, NH, DH]; weight, bias [NH * DH] or None.
    Differentiable; the gradient of h lies in memory as h does.
    """
    return layer_norm_op(h, weight, bias, eps, 1 if heads_first else 2)[0]
