"""The linear layer on int8 weights with a scale per output channel: the INT8 sibling of apply_fp8_linear, for symmetric
activations (what the reference's layer does, python/sglang/srt/layers/quantization/w8a8_int8.py: per_token_quant_int8, then
int8_scaled_mm) and for asymmetric ones, a scale and a zero point per token.  Asymmetric codes use all 256 steps on rows that
lie on one side of zero, as behind GELU, squared ReLU or a gate."""
from typing import Optional

import torch

from ..gemm import int8_scaled_mm, int8_scaled_mm_azp
from ..ops import _C


def int8_weight_sums(weight: torch.Tensor) -> torch.Tensor:
    """int32 [N]: the sums over K of an int8 weight, given as the column-major [K, N] view of its [N, K] rows.  What a
    product with zero points needs of the weight; made once, kept with it."""
    return _C.int8_weight_sums(weight)


def apply_int8_linear(
    input: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    weight_sums: Optional[torch.Tensor] = None,
    input_scale: Optional[torch.Tensor] = None,
    input_zero_point: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """input [..., K] times weight, the column-major [K, N] view of an int8 [N, K] parameter, weight_scale float32 with N
    elements or one.

    A half/bfloat16 input is quantised per token here, with zero points where `weight_sums` (int8_weight_sums(weight)) are given
    and without where not; the output has its dtype.  An int8 input is taken as quantised already (fused_rms_row_quant,
    silu_and_mul_row_quant, per_token_quant_int8 or per_token_quant_int8_asym): input_scale holds a value per token,
    input_zero_point too or None, and out_dtype says what the output is (bfloat16).  K % 16 == 0, N % 8 == 0; K <= 65536 with
    zero points.

    Rows that are not finite: with zero points a NaN or an infinity makes its whole output row NaN.  Without them the rows are
    quantised as per_token_quant_int8 does it, whose maximum skips a NaN: it counts as a zero and the output does not show it,
    while an infinity leaves no finite value in its output row.  (fused_rms_row_quant and silu_and_mul_row_quant show both in either form.)"""
    n = weight.shape[1]
    w_scale = weight_scale
    if w_scale.numel() == 1 and n != 1:
        w_scale = w_scale.reshape(-1).expand(n).contiguous()
    x = input.reshape(-1, input.shape[-1]) if input.dim() != 2 else input
    if input.dtype != torch.int8:
        if input_scale is not None or input_zero_point is not None:
            raise NotImplementedError("an input scale or zero point is only accepted with a pre-quantised int8 input")
        if out_dtype is not None and out_dtype != input.dtype:
            raise NotImplementedError("the output of a 16-bit input has the input's dtype")
        out = _C.int8_linear(x, weight, w_scale, weight_sums, bias)
    else:
        if input_scale is None:
            raise ValueError("an int8 input needs its input_scale")
        out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
        if input_zero_point is None:
            out = int8_scaled_mm(x, weight, input_scale, w_scale, out_dtype, bias)
        else:
            if weight_sums is None:
                raise ValueError("an input with zero points needs weight_sums")
            out = int8_scaled_mm_azp(x, weight, input_scale, w_scale, out_dtype, input_zero_point, weight_sums, bias)
    return out if input.dim() == 2 else out.view(*input.shape[:-1], n)
