"""Rows in 8 bits with one scale per token, fused with what produces them: the inputs of the row-scaled products
(apply_fp8_linear's and apply_int8_linear's GEMMs, the expert layer of a few tokens).  The siblings of
fused_rms_fp8_group_quant for whole rows; the reference runs its norm, its activation and its quantiser one after the other
(python/sglang/srt/layers/quantization/w8a8_int8.py, fp8_utils.py:1518-1559, layers/activation.py).

With y the row before its codes, all in float32 and not rounded on the way:

  float8_e4m3fn        scale = max|y| / 448, or `scale` where given;  code = e4m3(clamp(y / scale, -448, 448))
  int8                 scale = max(max|y|, 1e-10) / 127;  code = round(y / scale)
  int8, not symmetric  scale = max(hi - lo, 1e-10) / 255 with lo = min(0, min y), hi = max(0, max y);
                       zp = round(-128 - lo / scale);  code = clamp(round(y / scale) + zp, -128, 127)

The codes are (q, scale) or (q, scale, zp): q like the row, scale float32 [M, 1], zp int32 [M, 1]; y is about
scale * (q - zp).  A row of y that holds a NaN or an infinity gets a scale that is NaN or infinite; with a given scale a NaN stays
a NaN code and an infinity saturates (behind the norm the whole row is NaN).  Rows may have any length and alignment and lie any distance apart, or be one row
repeated (a stride of 0); rows that overlap otherwise raise.  Those of 8 to 32768 values are read once.  There is no gradient and
no torch.ops schema: under a tracer or a transform the functions raise NotImplementedError."""
from typing import Optional, Tuple

import torch

from ..ops import _C


def _codes(q, scale, zp):
    return (q, scale) if zp is None else (q, scale, zp)


def fused_rms_row_quant(
    inp: torch.Tensor,
    weight: torch.Tensor,
    epsilon: float,
    res: Optional[torch.Tensor] = None,
    dtype_quant: torch.dtype = torch.int8,
    symmetric: bool = True,
    scale: Optional[torch.Tensor] = None,
    output_unquantized: bool = False,
) -> Tuple[Tuple[torch.Tensor, ...], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(codes, y or None, inp + res or None) of y = v / sqrt(mean(v^2) + epsilon) * weight, v = inp + res.
    inp [M, N] half/bfloat16 with contiguous rows, res like inp, weight [N] float32 or of inp's dtype; y and inp + res are
    rounded to inp's dtype.  `scale`: one float32 on the device, float8_e4m3fn only (a static input scale); it comes back
    repeated for each row."""
    q, s, zp, y, res_out = _C.fused_rms_row_quant(inp, weight, epsilon, res, dtype_quant, symmetric, scale, output_unquantized)
    return _codes(q, s, zp), y, res_out


def silu_and_mul_row_quant(
    input: torch.Tensor,
    dtype_quant: torch.dtype = torch.int8,
    symmetric: bool = True,
    scale: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, ...]:
    """The codes of silu(gate) * up for rows of [gate | up], input [M, 2 * N] half/bfloat16 with contiguous rows: silu_and_mul
    and a per-token quantiser in one pass, without the rounding to 16 bits between them.  Gates below -87 give 0."""
    return _codes(*_C.silu_mul_row_quant(input, dtype_quant, symmetric, scale))
