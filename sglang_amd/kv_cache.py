"""Paged caches of keys and values: new tokens' rows into their slots, rotated and normalised on the way, in 16 or 8 bits, and the
rows of a context back in 16 bits.

A cache is [slots, heads, head size], or [pages, page size, heads, head size] in any order of memory with contiguous rows (a cache
that keeps the heads of a page together is passed transposed).  Slot s is row s % page size of page s / page size.  `slots` (int32
or int64, one per token) outside of the cache stand for no slot: padding, whose rows are not written, or read as zeros.  Slots that
are written in one call have to differ (of two tokens with the same slot, either may be kept, or parts of both, its codes with the
other one's scale among them).

A cache of the heads' dtype has no scale.  An 8-bit one holds, with y the row in float32:

  float8_e4m3fn, scale float32 [1], or [heads]     code = e4m3(clamp(y * (1 / scale), -448, 448)), the scale known beforehand
  float8_e4m3fn, scale float32 [slots..., heads]   scale = max|y| / 448 of the token's head, written to the slot's place
  int8, scale float32 [slots..., heads]            m = max(max|y|, 1e-10), scale = m / 127, code = round(y * (127 / m))

where [slots...] are the cache's own leading dimensions; a row that holds a NaN or an infinity gets a scale that is one.  1 / scale
and 127 / m are rounded to float32, as in the row quantisers: next to a tie a code may be the other one of the two.  A scale of
zero gives codes of zero; int8 rounds halves away from zero.  Rows beyond those of `slots` are left as they are, and their
scales too.

Memory that is written overlaps nothing else that a call is given.  There is no gradient and no torch.ops schema: under a tracer or a
transform the functions raise NotImplementedError."""
from typing import Optional, Sequence, Tuple

import torch

from .ops import _C


def append_kv(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    q: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    cos_sin: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    sections: Optional[Sequence[int]] = None,
    alternating: bool = False,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    epsilon: float = 1e-6,
    q_out: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """k and v [tokens, heads, head size] into their slots, in one launch with what else stands in front of the attention: k
    normalised by k_weight and rotated by positions and cos_sin where given, q (optional) alike by q_weight (rotary.py has the
    rotation, its axes and the norm).  Returns (q, k_out): the queries, new or in q_out, and k_out, which takes the keys that went
    into the cache in 16 bits (it may be k itself)."""
    return _C.append_kv(k, v, k_cache, v_cache, slots, k_scale, v_scale, q, positions, cos_sin, interleaved, sections, alternating, q_weight,
                        k_weight, epsilon, q_out, k_out)


def append_latent(
    latent: torch.Tensor,
    rope: torch.Tensor,
    latent_cache: torch.Tensor,
    rope_cache: torch.Tensor,
    slots: torch.Tensor,
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    weight: Optional[torch.Tensor] = None,
    epsilon: float = 1e-6,
    interleaved: bool = False,
    scale: Optional[torch.Tensor] = None,
    rope_scale: Optional[torch.Tensor] = None,
    q_rope: Optional[torch.Tensor] = None,
    q_out: Optional[torch.Tensor] = None,
) -> Optional[torch.Tensor]:
    """The two parts of a compressed row (multi-head latent attention) into their slots, in one launch: latent [tokens, C],
    normalised by `weight` where given, and rope [tokens, R], rotated; the queries' rotary parts q_rope [tokens, heads, R] are rotated
    alike and returned, new or in q_out.  The caches are [slots, C] and [slots, R], or paged, and may be views of the same rows.
    `scale` of an 8-bit latent_cache as above, or float32 [slots..., C / 128]: one per 128 values (C a multiple of 128;
    [slots..., 1]: per row).  rope_cache is in 16 bits, or in float8_e4m3fn with a given rope_scale."""
    return _C.append_latent(latent, rope, latent_cache, rope_cache, slots, positions, cos_sin, weight, epsilon, interleaved, scale, rope_scale,
                            q_rope, q_out)


def gather_kv(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slots: torch.Tensor,
    dtype: torch.dtype,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
    v_out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [len(slots), heads, head size] in `dtype` (half/bfloat16, a 16-bit cache's own): code * scale of the slots' rows, for
    attention over earlier tokens.  The same slot may be asked for more than once."""
    return _C.gather_kv(k_cache, v_cache, slots, dtype, k_scale, v_scale, k_out, v_out)


def gather_latent(
    latent_cache: torch.Tensor,
    rope_cache: torch.Tensor,
    slots: torch.Tensor,
    dtype: torch.dtype,
    scale: Optional[torch.Tensor] = None,
    rope_scale: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """[len(slots), C + R] in `dtype`: the two parts of the slots' compressed rows side by side."""
    return _C.gather_latent(latent_cache, rope_cache, slots, dtype, scale, rope_scale, out)
