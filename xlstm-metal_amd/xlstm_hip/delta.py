"""The gated delta rule on HIP: by chunks (``csrc/delta_*.hip``), token by token and one decode step.

For every head, with the state C [DHQK, DHV] (float32) and ``a = exp(g)``::

    C = a C + k (beta (v - (a C)^T k))^T,        h = scale C^T q

the matrix memory of the mLSTM with a correction in place of its input gate and normaliser: what C already answers to k is
taken off v before it is written.  Layouts are the chunkwise mLSTM kernels': q, k [B, NHK, S, DHQK], v [B, NH, S, DHV], g and
beta [B, NH, S], h [B, NH, S, DHV]; NH is a multiple of NHK, and head i of v reads head i // (NH / NHK) of q and k.  q, k, v share
a dtype (float32, bfloat16 or float16); g (log decay, at most 0; -inf starts afresh) and beta share one of their own.
``scale`` is DHQK ** -0.5 by default; DHQK up to 256.  q and k are taken as they are: norm them before.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

from torch import Tensor

from .ops import gated_delta_chunkwise_op, gated_delta_recurrent_op, gated_delta_step_inplace_op, gated_delta_step_op

__all__ = ["gated_delta_chunkwise", "gated_delta_recurrent", "gated_delta_step", "gated_delta_step_"]


def _scale(q: Tensor, scale: Optional[float]) -> float:
    return q.shape[-1] ** -0.5 if scale is None else float(scale)


def gated_delta_chunkwise(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, c_initial: Optional[Tensor] = None,
                          scale: Optional[float] = None,
                          return_last_states: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """h, or (h, C after the last token), for prompts and training: any S, on the matrix cores by chunks of 64 tokens.

    q, k and v are read in place where their last axis is contiguous (a projection's transposed views).  Tokens with g and
    beta 0 leave the state alone, whatever finite q, k and v they have: pad with them.  A value that is not finite spoils the h of
    its chunk from its first token on, one of v or of the state that of its own column only.
    """
    h, c = gated_delta_chunkwise_op(q, k, v, g, beta, c_initial, _scale(q, scale), return_last_states)
    return (h, c) if return_last_states else h


def gated_delta_recurrent(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, c_initial: Optional[Tensor] = None,
                          scale: Optional[float] = None,
                          return_last_states: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """``gated_delta_chunkwise`` token by token in float32, for a few tokens (drafted ones, say); forward only."""
    h, c = gated_delta_recurrent_op(q, k, v, g, beta, c_initial, _scale(q, scale), return_last_states)
    return (h, c) if return_last_states else h


def gated_delta_step(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, c: Tensor,
                     scale: Optional[float] = None) -> Tuple[Tensor, Tensor]:
    """One token, its tensors without the S axis: (h [B, NH, DHV], the new state); forward only."""
    return gated_delta_step_op(q, k, v, g, beta, c, _scale(q, scale))


def gated_delta_step_(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, c: Tensor,
                      scale: Optional[float] = None) -> Tuple[Tensor, Tensor]:
    """``gated_delta_step`` that updates c (float32, contiguous) in place: (h, c)."""
    return gated_delta_step_inplace_op(q, k, v, g, beta, c, _scale(q, scale)), c
