"""Rotary positions on the heads of queries and keys, with RMSNorm of every head in front of it where a model has one.

Heads are half/bfloat16 [tokens, heads, head size] with contiguous rows (views into a projection's output will do; head size even, at
most 1024).  cos_sin [positions, R], float32 or of the heads' dtype, at most 2 GiB, holds R / 2 cosines and then R / 2 sines per position, R
even and at most the head size.  Pair i < R / 2 of a head is (x[i], x[i + R / 2]), with `interleaved` (x[2 i], x[2 i + 1]); (a, b) becomes
(a cos - b sin, b cos + a sin) and the values behind the first R stay.

positions (int32 or int64) is [tokens], or [axes, tokens] with `sections`, how many pairs turn by each of up to four axes (the time,
height and width of an image or video): the first sections[0] pairs by axis 0, the next sections[1] by axis 1 and so on; with
`alternating`, pair i by axis i % axes where i < axes * sections[i % axes] and by axis 0 otherwise.  A position outside of the
table gives NaN.

All arithmetic is in float32, rounded once.  Outputs are new tensors, or q_out and k_out where given: they may be q and k themselves,
and overlap nothing else.  There is no gradient and no torch.ops schema: under a tracer or a transform the functions raise
NotImplementedError."""
from typing import Optional, Sequence, Tuple

import torch

from .ops import _C


def rotate_qk(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    interleaved: bool = False,
    sections: Optional[Sequence[int]] = None,
    alternating: bool = False,
    q_out: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(q, k) rotated, in one launch.  k may have a head count and size of its own, or be None."""
    return _C.rotate_qk(q, k, positions, cos_sin, interleaved, sections, alternating, q_out, k_out)


def norm_rotate_qk(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    epsilon: float,
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    interleaved: bool = False,
    sections: Optional[Sequence[int]] = None,
    alternating: bool = False,
    q_out: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """rotate_qk of the normalised heads x / sqrt(mean(x^2) + epsilon) * weight, the weights [head size] float32 or of the heads'
    dtype.  A head whose sum of squares is not finite in float32 is NaN; with an epsilon of zero, values below 1e-19, whose squares are
    below float32's normal range, lose digits."""
    return _C.norm_rotate_qk(q, k, q_weight, k_weight, epsilon, positions, cos_sin, interleaved, sections, alternating, q_out, k_out)
