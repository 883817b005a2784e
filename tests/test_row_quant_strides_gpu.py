"""Row strides of the operators that quantise rows: from the row's length up, or 0; rows that overlap otherwise are refused."""
import pytest
import torch

from . import row_layers as rl

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden", [64, 1000, 8191])
def test_strides(dev, hidden):
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant, silu_and_mul_row_quant
    from sglang_amd.quantization.int8_kernel import per_token_quant_int8_asym

    line = torch.randn(24 * hidden, generator=torch.Generator().manual_seed(hidden)).to(torch.bfloat16).to(dev)
    w = torch.ones(hidden, device=dev)

    def calls(x, wide, res=None):
        return (lambda: fused_rms_row_quant(x, w, 1e-6, res=x if res is None else res)[0], lambda: silu_and_mul_row_quant(wide), lambda: per_token_quant_int8_asym(x))

    for stride in (0, hidden, hidden + 1, 3 * hidden):
        x, wide = line.as_strided((4, hidden), (stride, 1)), line.as_strided((4, 2 * hidden), (2 * stride, 1))
        for got, want in zip(calls(x, wide), calls(x.contiguous(), wide.contiguous())):
            got, want = got(), want()
            # (unaligned rows add up in another order behind a norm, so both are off by what their sums are)
            assert torch.allclose(got[1], want[1], rtol=2 * (rl.rms_error(hidden) + 8 * rl.U), atol=0)
            assert (got[0].int() - want[0].int()).abs().max() <= 1
    for stride in (1, 8, hidden - 1):
        x, wide = line.as_strided((4, hidden), (stride, 1)), line.as_strided((4, 2 * hidden), (stride, 1))
        for call in calls(x, wide):
            with pytest.raises(RuntimeError, match="stride"):
                call()
        with pytest.raises(RuntimeError, match="stride"):
            calls(x.contiguous(), wide, x)[0]()
        one = x[:1]  # (one row has no stride)
        assert torch.equal(per_token_quant_int8_asym(one)[0], per_token_quant_int8_asym(one.contiguous())[0])
