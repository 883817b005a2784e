"""The expert layer of a few tokens in two launches, on rows that are in 8 bits already.

In a decode step the norm in front of the experts hands over codes and scales (quantization.fused_row_quant) beside the 16-bit
row that the router reads, so the layer has nothing to quantise or sort in front of its first product: pairs that share an
expert are found inside the kernels, and the sum over a token's experts ends the second one.  The general layer
(fused_experts; python/sglang/srt/layers/moe/moe_runner/triton_utils/fused_moe.py:401-785) takes 16-bit rows and any number of them.

Which of the two: the general one reads an expert's weights once; this one once for every pass over the rows that meet it, of one row at one
token, two at two, else four, and fewer where eight waves' rows of I codes do not fit 64 KB (from eight pairs on two beyond I = 2048, one beyond
4096) or sixteen waves share the second launch (two).  Int8, us, quantiser included, here | fused_experts: 128 experts of 2048 x 768, 8 each,
1 / 4 / 8 tokens 16 | 30, 33 | 49, 53 | 63; 64 of 4096 x 1536, 8 each, 1 / 4 / 8 34 | 48, 90 | 101, 149 | 160; 8 of 4096 x 1536, 2 each, 4 / 8 / 16 / 32
26 | 37, 34 | 39, 58 | 49, 78 | 50; 16 of 4096 x 4096, 2 each, 1 / 4 / 8 / 16 34 | 40, 81 | 80, 117 | 102, 193 | 117; 8 of 4096 x 14336, 2 each,
1 / 4 / 8 101 | 74, 275 | 185, 603 | 233.  So: this one for I up to 2048 while experts meet up to two or three rows each, up to 4096 at about
one row each, the general one otherwise."""
from typing import Optional

import torch

from ..ops import _C

MAX_PAIRS = 64


def takes_few_tokens(num_tokens: int, topk: int) -> bool:
    """Whether fused_experts_few_tokens takes so many tokens and experts per token (not whether it is faster than fused_experts
    on them: the head of this file has the times)."""
    return num_tokens * topk <= MAX_PAIRS


def fused_experts_few_tokens(
    hidden_q: torch.Tensor,
    hidden_scale: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    w1_scale: torch.Tensor,
    w2_scale: torch.Tensor,
    topk_weights: torch.Tensor,
    topk_ids: torch.Tensor,
    out_dtype: torch.dtype = torch.bfloat16,
    b1: Optional[torch.Tensor] = None,
    b2: Optional[torch.Tensor] = None,
    routed_scaling_factor: Optional[float] = None,
) -> torch.Tensor:
    """[M, H] of gated-SiLU experts: hidden_q [M, H] float8_e4m3fn or int8 (symmetric codes) with hidden_scale float32 (one per
    token), w1 [E, 2 * I, H] and w2 [E, H, I] of that dtype, w1_scale / w2_scale one float32 per output channel, b1 / b2 one
    value per output channel in out_dtype, topk_weights and topk_ids [M, topk].  Pairs whose id is outside [0, E) contribute
    nothing.  Between the products the rows stay in float32 and are quantised per (token, expert) pair by the formulas of
    fused_row_quant; the output is rounded once.  H, I multiples of 16, H <= 32768, I <= 16384; more than MAX_PAIRS pairs raise
    NotImplementedError (fused_experts takes them)."""
    return _C.experts_few_tokens(hidden_q, hidden_scale, w1, w2, w1_scale, w2_scale, topk_weights, topk_ids, out_dtype, b1, b2,
                                 1.0 if routed_scaling_factor is None else routed_scaling_factor)
