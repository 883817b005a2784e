"""Rows to 8-bit codes at the ends of what the types hold."""
import pytest
import torch

from . import row_layers as rl

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden", [16, 512, 1000, 4096, 8192, 33024, 333])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_span_beyond_float32(dev, hidden, dtype):
    """hi - lo of finite values may be twice the largest float32; the scale is a 255th of it and finite."""
    from sglang_amd.quantization.int8_kernel import per_token_quant_int8_asym

    g = torch.Generator().manual_seed(hidden)
    x = torch.randn(5, hidden, generator=g) * 1e38
    x = x.clamp(-3.3e38, 3.3e38).to(dtype)
    top = torch.finfo(dtype).max
    x[0, 1], x[0, hidden - 1] = top, -top  # a mask's value and its opposite
    x[1, 0], x[1, hidden // 2] = 3e38, -2e38
    x[2, 3] = -top  # on one side of zero: no overflow
    x[2] = -x[2].abs()
    x[3] = x[3] * 1e-38
    q, s, zp = per_token_quant_int8_asym(x.to(dev))
    rl.check_codes(x.double(), 0.0, (q), s, zp)
    # what is not finite still is not
    x[4, 5] = float("inf")
    s = per_token_quant_int8_asym(x.to(dev))[1].cpu().view(-1)
    assert torch.isfinite(s).tolist() == [True, True, True, True, False]


@pytest.mark.parametrize("m", [1, 3, 16, 17, 80])
def test_a_linear_of_such_rows(dev, m):
    """In one launch and in two: the bits of its quantiser and its product, finite where the weight's scale is small enough."""
    from sglang_amd import int8_scaled_mm_azp
    from sglang_amd.quantization.int8_kernel import per_token_quant_int8_asym
    from sglang_amd.quantization.int8_utils import apply_int8_linear, int8_weight_sums

    g = torch.Generator().manual_seed(m)
    n, k = 256, 1024
    x = torch.randn(m, k, generator=g).to(torch.bfloat16).to(dev)
    x[m // 2, 7], x[m // 2, k - 9] = 3e38, -3e38
    w = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8).to(dev)
    ws = torch.full((n,), 1e-10, device=dev)
    sums = int8_weight_sums(w.t())
    out = apply_int8_linear(x, w.t(), ws, sums)
    q, s, zp = per_token_quant_int8_asym(x)
    assert torch.isfinite(out).all() and torch.equal(out, int8_scaled_mm_azp(q, w.t(), s, ws, torch.bfloat16, zp, sums))
    rl.check_product(out, q, zp, w, s, ws, None)


@pytest.mark.parametrize("hidden", [64, 1024, 8192])
def test_a_norm_and_a_silu_of_such_a_span(dev, hidden):
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant, silu_and_mul_row_quant

    g = torch.Generator().manual_seed(hidden)
    x = torch.randn(2, hidden, generator=g).clamp(-2, 2)
    x[:, 3], x[:, 5] = 1.0, -1.0
    x = x.to(torch.bfloat16)
    w = torch.ones(hidden)
    w[3] = w[5] = 2e38
    codes, _, _ = fused_rms_row_quant(x.to(dev), w.to(dev), 1e-6, symmetric=False)
    y = rl.rms(x, w, 1e-6)[1]
    assert (y[:, 3] - y[:, 5] > 3.5e38).all()
    rl.check_codes(y, rl.rms_error(hidden), *codes)
    gate = torch.full_like(x, 4.0)
    up = x.clone()
    up[:, 3], up[:, 5] = 7e37, -7e37
    xx = torch.cat([gate, up], dim=1)
    xx[1, 5] = -0.5  # the one row on both sides, the other on one
    y = rl.silu_mul(xx)
    rl.check_codes(y, rl.silu_error(xx), *silu_and_mul_row_quant(xx.to(dev), symmetric=False))
