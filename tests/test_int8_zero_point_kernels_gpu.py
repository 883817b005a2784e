"""Products with zero points on the kernels and at the ends of the range that test_int8_asym_gpu.py does not reach."""
import pytest
import torch

from . import row_layers as rl
from .test_int8_asym_gpu import STREAMING, WIDE, _operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(17, 200, 48), (24, 4096, 16), (32, 1000, 496), (33, 520, 144), (40, 264, 400), (48, 24, 16), (64, 4096, 272), (64, 10240, 112)])
@pytest.mark.parametrize("dtype,with_bias", [(torch.bfloat16, False), (torch.float16, True)])
def test_a_short_ragged_sum_at_17_to_64_rows(dev, m, n, k, dtype, with_bias):
    from sglang_amd import int8_scaled_mm, int8_scaled_mm_azp
    from sglang_amd._lib import lib
    from sglang_amd.quantization.int8_utils import int8_weight_sums

    a, w, zp, sa, sb, bias = _operands(dev, m, n, k, m + n + k)
    if dtype == torch.float16:
        sa, sb = sa * 2.0 ** -6, sb * 2.0 ** -4
    bias = bias.to(dtype) if with_bias else None
    sums = int8_weight_sums(w.t())
    print(f"asymmetric int8 {m} x {n} x {k}", flush=True)
    rl.check_product(int8_scaled_mm_azp(a, w.t(), sa, sb, dtype, zp, sums, bias), a, zp, w, sa, sb, bias)
    none = int8_scaled_mm_azp(a, w.t(), sa, sb, dtype, torch.zeros_like(zp), sums, bias)
    ran = lib.sglamd_last_gemm_kernel()
    assert ran == STREAMING
    assert torch.equal(none, int8_scaled_mm(a, w.t(), sa, sb, dtype, bias)) and ran == lib.sglamd_last_gemm_kernel()


@pytest.mark.parametrize("m,n,k,tiles", [(64, 16452, 14848, 6), (40, 49348, 22528, 8), (33, 65796, 20992, 9)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_wide_streaming_form_without_scratch(dev, m, n, k, tiles, dtype):
    """33 to 64 rows where strips would split K and have no slabs for it: sampled blocks of weight rows."""
    from sglang_amd._lib import lib

    if dtype == torch.float16 and tiles != 6:
        pytest.skip("fp16 output covered on one shape")
    g = torch.Generator(device=dev).manual_seed(m + n + k)
    a, w = (torch.randint(-128, 128, (rows, k), generator=g, device=dev, dtype=torch.int8) for rows in (m, n))
    zp = torch.randint(-128, 128, (m, 1), generator=g, device=dev, dtype=torch.int32)
    sa, sb = (torch.rand(rows, generator=g, device=dev) * 1e-3 + 1e-4 for rows in (m, n))
    bias = torch.randn(n, generator=g, device=dev).to(dtype) * 10
    sums = w.sum(dim=1, dtype=torch.int32)
    out = torch.empty(m, n, dtype=dtype, device=dev)
    print(f"wide, zero points M={m} N={n} K={k} {dtype}", flush=True)
    rc = lib.sglamd_int8_scaled_mm_azp(a.data_ptr(), k, w.data_ptr(), k, sa.data_ptr(), sb.data_ptr(), zp.data_ptr(), sums.data_ptr(), bias.data_ptr(),
                                       out.data_ptr(), n, 2 if dtype == torch.bfloat16 else 1, m, n, k, 0, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and lib.sglamd_last_gemm_kernel() == WIDE
    assert lib.sglamd_last_streaming_shape() >> 8 & 0xFF == tiles
    for at in (0, 128, n // 3, n // 2, n - 256, n - 100):
        part = slice(at, min(at + 128, n))
        rl.check_product(out[:, part], a, zp, w[part], sa, sb[part], bias[part])


@pytest.mark.parametrize("m,n", [(1, 64), (2, 64), (16, 512), (17, 64), (40, 256), (64, 1024), (100, 256), (130, 256), (300, 512)])
@pytest.mark.parametrize("a,w,zp", [(127, -128, -128), (-128, -128, 127), (127, 127, -128), (-128, 127, 127), (-128, -128, -383), (127, -128, 257)])
def test_the_ends_of_the_range(dev, m, n, a, w, zp):
    """K = 65536 equal factors, differences of either sign near 2^31.  With int8 zero points the products' sum and the zero point's part stay
    below 2^30 + 2^23; zero points of -383 and 257 make the second of them 383 * 2^23 and -257 * 2^23, which 32 bits do not hold, and the difference
    fits again."""
    from sglang_amd import int8_scaled_mm_azp
    from sglang_amd.quantization.int8_utils import int8_weight_sums

    k = 65536
    want = k * (a - zp) * w
    assert -2 ** 31 <= want < 2 ** 31
    at, wt = torch.full((m, k), a, device=dev, dtype=torch.int8), torch.full((n, k), w, device=dev, dtype=torch.int8)
    z, one = torch.full((m, 1), zp, device=dev, dtype=torch.int32), torch.ones(max(m, n), device=dev)
    out = int8_scaled_mm_azp(at, wt.t(), one[:m], one[:n], torch.bfloat16, z, int8_weight_sums(wt.t()))
    # (the sum is converted to float32, then to the output's type)
    assert (out.cpu() == torch.tensor(float(want), dtype=torch.float64).float().to(torch.bfloat16)).all()
