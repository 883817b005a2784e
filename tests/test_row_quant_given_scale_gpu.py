"""e4m3 rows with a given scale: what becomes of a NaN and of an infinity, value by value."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
SCALE = 0.011
# (a wave, workgroups of several sizes, pieces that overlap, the value-by-value form on either side)
HIDDEN = [5, 64, 333, 1024, 4096, 8192, 8191, 16384, 20000, 32776]


def _rows(g, *shape):
    return (torch.randn(*shape, generator=g) * 2).to(torch.bfloat16)


def _codes(pair):
    return pair[0].cpu().float()


@pytest.mark.parametrize("hidden", HIDDEN)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_norm_of_a_bad_row_is_all_nan(dev, hidden, bad):
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant

    x, w = _rows(torch.Generator().manual_seed(hidden), 4, hidden), torch.ones(hidden)
    scale = torch.full((1,), SCALE, device=dev)
    for residual in (False, True):
        clean = fused_rms_row_quant(x.to(dev), w.to(dev), 1e-6, res=x.to(dev) if residual else None, dtype_quant=F8, scale=scale)[0]
        spoilt = x.clone()
        spoilt[2, hidden // 2 + 1] = bad
        rows = (x, spoilt) if residual else (spoilt, None)
        got = fused_rms_row_quant(rows[0].to(dev), w.to(dev), 1e-6, res=None if rows[1] is None else rows[1].to(dev), dtype_quant=F8, scale=scale)[0]
        assert not _codes(clean).isnan().any()
        assert _codes(got)[2].isnan().all()
        others = [0, 1, 3]
        assert torch.equal(_codes(got)[others], _codes(clean)[others])
        assert (got[1].cpu() == torch.tensor(SCALE)).all()


@pytest.mark.parametrize("hidden", HIDDEN)
@pytest.mark.parametrize("where", ["gate", "up"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_silu_spoils_the_one_value(dev, hidden, where, bad):
    """A NaN stays a NaN code, so does a gate of -inf (-inf times 0); an infinity saturates with its sign.  All other codes are
    those of the row without it."""
    from sglang_amd.quantization.fused_row_quant import silu_and_mul_row_quant

    x = _rows(torch.Generator().manual_seed(hidden), 4, 2 * hidden)
    at = hidden // 2 + 1
    x[2, at], x[2, hidden + at] = -0.5, -0.25  # what stands beside the bad value is not zero
    scale = torch.full((1,), SCALE, device=dev)
    clean = _codes(silu_and_mul_row_quant(x.to(dev), dtype_quant=F8, scale=scale))
    x[2, at if where == "gate" else hidden + at] = bad
    got = silu_and_mul_row_quant(x.to(dev), dtype_quant=F8, scale=scale)
    codes = _codes(got)
    if bad != bad or (where == "gate" and bad < 0):
        assert codes[2, at].isnan()
    else:
        # gate +inf times an up of -0.25; silu(-0.5) < 0 times an up of either sign
        assert codes[2, at] == (-448 if bad > 0 else 448)
    codes[2, at] = clean[2, at]
    assert torch.equal(codes, clean) and not clean.isnan().any()
    assert (got[1].cpu() == torch.tensor(SCALE)).all()
