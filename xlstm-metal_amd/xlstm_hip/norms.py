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
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dim() != 1 or x.dim() < 1 or t.shape[0] != x.shape[-1]):
            raise ValueError(f"layer_norm: {name} must be ({x.shape[-1] if x.dim() else '?'},), got {tuple(t.shape)}")
    return layer_norm_op(x, weight, bias, float(eps))[0]


def multi_head_layer_norm(h: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-6,
                          heads_first: bool = True) -> Tensor:
    """Layer norm of every head over DH, as [B, S, NH * DH].

    h is [B, NH, S, DH] (``heads_first``, the chunkwise output) or [B, S, NH, DH]; weight, bias [NH * DH] or None.
    Differentiable; the gradient of h lies in memory as h does.
    """
    if h.dim() != 4:
        raise ValueError(f"multi_head_layer_norm: h must be 4-D, got {tuple(h.shape)}")
    x = h.transpose(1, 2) if heads_first else h
    B, S, NH, DH = x.shape
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dim() != 1 or t.shape[0] != NH * DH):
            raise ValueError(f"multi_head_layer_norm: {name} must be ({NH * DH},), got {tuple(t.shape)}")
    w, b = (None if t is None else t.view(NH, DH) if t.is_contiguous() else t.reshape(NH, DH) for t in (weight, bias))
    return layer_norm_op(x, w, b, float(eps))[0].view(B, S, NH * DH)
