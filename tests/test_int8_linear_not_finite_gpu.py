"""What the symmetric int8 linear makes of rows that are not finite: as its text says, and as per_token_quant_int8 quantises them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(1, 256, 1024), (16, 512, 2048), (17, 256, 512), (64, 2048, 1024), (300, 512, 400)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_nan_counts_as_zero_and_an_infinity_spoils_its_row(dev, m, n, k, dtype):
    from sglang_amd.quantization.int8_utils import apply_int8_linear, int8_weight_sums

    g = torch.Generator().manual_seed(m + k)
    x = torch.randn(m, k, generator=g).to(dtype).to(dev)
    w = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8).to(dev)
    ws = torch.rand(n, generator=g).to(dev) * 1e-4 + 1e-5
    row, others = m // 2, [r for r in range(m) if r != m // 2]
    zero, nan, inf = x.clone(), x.clone(), x.clone()
    zero[row, k // 3], nan[row, k // 3], inf[row, k // 3] = 0.0, float("nan"), float("-inf")
    want = apply_int8_linear(zero, w.t(), ws)
    assert torch.isfinite(want).all()
    assert torch.equal(apply_int8_linear(nan, w.t(), ws), want)
    out = apply_int8_linear(inf, w.t(), ws)
    assert not torch.isfinite(out[row]).any() and torch.equal(out[others], want[others])
    # with zero points both are visible
    for bad in (nan, inf):
        out = apply_int8_linear(bad, w.t(), ws, int8_weight_sums(w.t()))
        assert out[row].isnan().all() and torch.isfinite(out[others]).all()
