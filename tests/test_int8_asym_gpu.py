"""Products of int8 rows with a scale and a zero point each, and the linear layer on top, against exact integers."""
import pytest
import torch

from . import row_layers as rl

pytestmark = pytest.mark.gpu
STREAMING, TILE64, TILE128, TILE256, GENERIC, WIDE, TILE192, STRIP = 1, 2, 3, 4, 6, 8, 9, 10
TILES = (TILE64, TILE128, TILE256, TILE192)


def _operands(dev, m, n, k, seed, pitch=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(-128, 128, (m, k + pitch), generator=g, dtype=torch.int8)[:, :k]
    w = torch.randint(-128, 128, (n, k + pitch), generator=g, dtype=torch.int8)[:, :k]
    zp = torch.randint(-128, 128, (m, 1), generator=g, dtype=torch.int32)
    sa, sb = torch.rand(m, 1, generator=g) * 1e-2 + 1e-3, torch.rand(n, 1, generator=g) * 1e-2 + 1e-3
    bias = torch.randn(n, generator=g) * 50
    return [t.to(dev) for t in (a, w, zp, sa, sb, bias)]


# every kernel that a dense int8 product may run, every row count of their epilogues, ragged sizes
SIZES = [
    (1, 512, 512, STREAMING), (1, 8, 16, STREAMING), (5, 2048, 7168, STREAMING), (16, 1000, 400, STREAMING), (17, 2048, 2048, STREAMING),
    (32, 4096, 4096, STREAMING), (40, 256, 512, STREAMING), (64, 512, 512, None), (24, 40000, 4096, STRIP), (48, 28672, 4096, STRIP),
    (80, 28672, 4096, STRIP), (97, 28672, 4096, STRIP), (128, 28672, 4096, STRIP), (128, 57344, 2048, None), (120, 7168, 16384, None),
    (100, 20480, 8192, None), (64, 8192, 28672, None), (130, 4096, 4096, None), (200, 8192, 8192, None), (300, 2048, 2048, None),
    (300, 8192, 28672, None), (700, 8192, 1024, None), (512, 36864, 1024, None), (1100, 4096, 1536, None), (2048, 8192, 512, None),
    (100, 8192, 4112, None), (300, 264, 4112, None),
    # a short K that ends inside a K block: one block, the first of two, the fourth
    (65, 24, 48, TILE64), (130, 200, 400, TILES), (1000, 8304, 16, TILES), (65, 1000, 112, TILE64), (257, 520, 144, TILES), (300, 4096, 496, TILES),
    (2000, 3000, 64, TILES), (4096, 264, 272, TILES),
]


@pytest.mark.parametrize("m,n,k,kernel", SIZES)
@pytest.mark.parametrize("dtype,with_bias", [(torch.bfloat16, False), (torch.float16, True)])
def test_product(dev, m, n, k, kernel, dtype, with_bias):
    from sglang_amd import int8_scaled_mm, int8_scaled_mm_azp
    from sglang_amd._lib import lib
    from sglang_amd.quantization.int8_utils import int8_weight_sums

    a, w, zp, sa, sb, bias = _operands(dev, m, n, k, m + n + k)
    if dtype == torch.float16:
        sa, sb = sa * 2.0 ** -6, sb * 2.0 ** -4  # results that a half holds
    bias = bias.to(dtype) if with_bias else None
    print(f"asymmetric int8 {m} x {n} x {k}", flush=True)
    sums = int8_weight_sums(w.t())
    out = int8_scaled_mm_azp(a, w.t(), sa, sb, dtype, zp, sums, bias)
    ran = lib.sglamd_last_gemm_kernel()
    rl.check_product(out, a, zp, w, sa, sb, bias)
    # without zero points it is the symmetric product, on the same kernel to the bit (a short ragged K has another one there)
    none = int8_scaled_mm_azp(a, w.t(), sa, sb, dtype, torch.zeros_like(zp), sums, bias)
    rl.check_product(none, a, None, w, sa, sb, bias)
    symmetric = int8_scaled_mm(a, w.t(), sa, sb, dtype, bias)
    assert ran == lib.sglamd_last_gemm_kernel() or (k < 512 and k % 128)
    if ran == lib.sglamd_last_gemm_kernel():
        assert torch.equal(none, symmetric)
    if kernel is not None:
        assert ran in (kernel if isinstance(kernel, tuple) else (kernel,)), f"ran kernel {ran}, meant for {kernel}"
    # in the same bits on every run
    assert torch.equal(out, int8_scaled_mm_azp(a, w.t(), sa, sb, dtype, zp, sums, bias))


def test_all_kernels_are_among_the_sizes(dev):
    from sglang_amd import int8_scaled_mm_azp
    from sglang_amd._lib import lib

    ran = set()
    for m, n, k, _ in SIZES:
        a, w = torch.zeros(m, k, device=dev, dtype=torch.int8), torch.zeros(n, k, device=dev, dtype=torch.int8)
        s = torch.ones(max(m, n), device=dev)
        i = torch.zeros(max(m, n), device=dev, dtype=torch.int32)
        out = int8_scaled_mm_azp(a, w.t(), s[:m], s[:n], torch.bfloat16, i[:m], i[:n])
        assert not out.any()
        ran.add(lib.sglamd_last_gemm_kernel())
    assert ran >= {STREAMING, TILE64, TILE128, TILE256, TILE192, STRIP}, ran


@pytest.mark.parametrize("k", [48, 528])
def test_rows_further_apart_than_32_bits_reach(dev, k):
    """The generic kernel, which alone addresses operands beyond 2 GiB: 70 rows of them, 32 MB apart."""
    from sglang_amd import int8_scaled_mm_azp
    from sglang_amd._lib import lib
    from sglang_amd.quantization.int8_utils import int8_weight_sums

    _, w, zp, sa, sb, _ = _operands(dev, 70, 136, k, k)
    a = torch.randint(-128, 128, (70, k), dtype=torch.int8, device=dev)
    far = torch.empty(70 << 25, dtype=torch.int8, device=dev).as_strided((70, k), (1 << 25, 1)).copy_(a)
    sums = int8_weight_sums(w.t())
    out = int8_scaled_mm_azp(far, w.t(), sa, sb, torch.bfloat16, zp, sums)
    assert lib.sglamd_last_gemm_kernel() == GENERIC
    assert torch.equal(out, int8_scaled_mm_azp(a, w.t(), sa, sb, torch.bfloat16, zp, sums))


def test_the_largest_sums(dev):
    """Every factor at its end of the range over the longest K: the difference fills 31 bits while its parts wrap."""
    from sglang_amd import int8_scaled_mm_azp
    from sglang_amd.quantization.int8_utils import int8_weight_sums

    k = 65536
    for m, n in ((2, 64), (130, 256)):
        a = torch.full((m, k), 127, device=dev, dtype=torch.int8)
        w = torch.full((n, k), -128, device=dev, dtype=torch.int8)
        zp = torch.full((m, 1), -128, device=dev, dtype=torch.int32)
        one = torch.ones(max(m, n), device=dev)
        out = int8_scaled_mm_azp(a, w.t(), one[:m], one[:n], torch.bfloat16, zp, int8_weight_sums(w.t()))
        assert (out.double() == float(torch.tensor(-255.0 * 128 * k).to(torch.bfloat16))).all()
    with pytest.raises(NotImplementedError):
        a, w = torch.zeros(1, k + 16, device=dev, dtype=torch.int8), torch.zeros(8, k + 16, device=dev, dtype=torch.int8)
        int8_scaled_mm_azp(a, w.t(), one[:1], one[:8], torch.bfloat16, zp[:1], torch.zeros(8, device=dev, dtype=torch.int32))


@pytest.mark.parametrize("m,n,k,pitch", [(3, 512, 1024, 16), (40, 1024, 512, 128), (300, 512, 1024, 32)])
def test_operands_with_a_pitch_and_sums_off_16_bytes(dev, m, n, k, pitch):
    from sglang_amd import int8_scaled_mm_azp
    from sglang_amd.quantization.int8_utils import int8_weight_sums

    a, w, zp, sa, sb, bias = _operands(dev, m, n, k, m, pitch)
    shifted = [torch.cat([t.view(-1)[:1], t.view(-1)])[1:] for t in (zp, int8_weight_sums(w.t()), sa, sb, bias.bfloat16())]
    assert shifted[1].data_ptr() % 16
    out = int8_scaled_mm_azp(a, w.t(), shifted[2], shifted[3], torch.bfloat16, shifted[0], shifted[1], shifted[4])
    rl.check_product(out, a, zp, w, sa, sb, bias.bfloat16())


@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (1, 64, 16), (7, 1000, 4096), (33, 2048, 2048), (300, 512, 4112)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
def test_linear(dev, m, n, k, dtype, asym, with_bias):
    """The layer is its quantiser and its product, to the bit."""
    from sglang_amd import int8_scaled_mm, int8_scaled_mm_azp
    from sglang_amd.quantization.int8_kernel import per_token_quant_int8, per_token_quant_int8_asym
    from sglang_amd.quantization.int8_utils import apply_int8_linear, int8_weight_sums

    g = torch.Generator().manual_seed(m + n)
    x = torch.nn.functional.gelu(torch.randn(m, k, generator=g) * 2).to(dtype).to(dev)
    _, w, _, _, sb, bias = _operands(dev, m, n, k, m)
    sb = sb * 0.01
    bias = (bias / 50).to(dtype) if with_bias else None
    sums = int8_weight_sums(w.t()) if asym else None
    out = apply_int8_linear(x, w.t(), sb, weight_sums=sums, bias=bias)
    if asym:
        q, s, zp = per_token_quant_int8_asym(x)
        steps = int8_scaled_mm_azp(q, w.t(), s, sb, dtype, zp, sums, bias)
        rl.check_product(out, q, zp, w, s, sb, bias)
        taken = apply_int8_linear(q, w.t(), sb, weight_sums=sums, input_scale=s, input_zero_point=zp, bias=bias, out_dtype=dtype)
    else:
        q, s = per_token_quant_int8(x)
        steps = int8_scaled_mm(q, w.t(), s, sb, dtype, bias)
        taken = apply_int8_linear(q, w.t(), sb, input_scale=s, bias=bias, out_dtype=dtype)
    assert torch.equal(out, steps) and torch.equal(out, taken)
    assert torch.equal(apply_int8_linear(x.view(1, m, k), w.t(), sb, weight_sums=sums, bias=bias), out.view(1, m, n))


@pytest.mark.parametrize("n,k", [(64, 128), (1024, 256), (7168, 16384), (2112, 7168), (24576, 1536), (576, 4096), (36864, 640), (4160, 2432), (264, 2064)])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 12, 16])
@pytest.mark.parametrize("asym", [False, True])
@pytest.mark.parametrize("dtype,with_bias", [(torch.bfloat16, False), (torch.float16, True)])
def test_linear_of_a_few_rows_quantised_in_the_product(dev, m, n, k, asym, dtype, with_bias):
    """The row's extremes span all of its pieces, several waves and passes; rows on one side of zero, of zeros, with a NaN or an
    infinity; a view into longer rows."""
    from sglang_amd import int8_scaled_mm, int8_scaled_mm_azp
    from sglang_amd.quantization.int8_kernel import per_token_quant_int8, per_token_quant_int8_asym
    from sglang_amd.quantization.int8_utils import apply_int8_linear, int8_weight_sums

    g = torch.Generator(device=dev).manual_seed(m + n + k)
    w = torch.randint(-128, 128, (n, k), generator=g, device=dev, dtype=torch.int8)
    ws = torch.rand(n, 1, generator=g, device=dev) * 1e-4 + 1e-5
    b = torch.randn(n, generator=g, device=dev).to(dtype) if with_bias else None
    sums = int8_weight_sums(w.t()) if asym else None
    for kind in ("plain", "zeros", "one side", "nan", "inf", "view"):
        x = torch.randn(m, k + (64 if kind == "view" else 0), generator=g, device=dev).to(dtype)
        x[-1, k - 1] = 50.0  # the extreme of a row in its last piece
        if kind == "zeros":
            x[0] = 0
        elif kind == "one side":
            x = -x.abs() - 1
        elif kind == "nan":
            x[m // 2, k // 2] = float("nan")
        elif kind == "inf":
            x[m // 2, 3] = float("-inf")
        elif kind == "view":
            x = x[:, :k]
        print(f"one launch, int8, M={m} N={n} K={k} {dtype} {kind}", flush=True)
        out = apply_int8_linear(x, w.t(), ws, sums, bias=b)
        if asym:
            q, s, zp = per_token_quant_int8_asym(x)
            ref = int8_scaled_mm_azp(q, w.t(), s, ws, dtype, zp, sums, b)
        else:
            q, s = per_token_quant_int8(x.contiguous())
            ref = int8_scaled_mm(q, w.t(), s, ws, dtype, b)
        assert torch.equal(out.isnan(), ref.isnan())
        assert torch.equal(out.nan_to_num(), ref.nan_to_num())
        if asym and kind in ("nan", "inf"):
            assert out[m // 2].isnan().all() and out.isnan().any(dim=1).sum() == 1


def test_linear_of_views_one_scale_and_no_rows(dev):
    from sglang_amd.quantization.int8_utils import apply_int8_linear, int8_weight_sums

    g = torch.Generator().manual_seed(9)
    wide = torch.randn(6, 3000, generator=g).to(torch.bfloat16).to(dev)
    _, w, _, _, sb, _ = _operands(dev, 6, 64, 1024, 4)
    sums = int8_weight_sums(w.t())
    for view in (wide[:, 8:1032], wide[:, 1:1025], wide[::2, :1024]):
        for asym in (None, sums):
            assert torch.equal(apply_int8_linear(view, w.t(), sb, asym), apply_int8_linear(view.contiguous(), w.t(), sb, asym))
    line = wide.view(-1)
    for view in (wide[:1, :1024].expand(5, 1024), line.as_strided((4, 1024), (8, 1)), line.as_strided((1, 1024), (1, 1)), wide[:1, :1024].expand(40, 1024)):
        for asym in (None, sums):
            assert torch.equal(apply_int8_linear(view, w.t(), sb, asym), apply_int8_linear(view.contiguous(), w.t(), sb, asym))
    one = torch.full((1,), 0.01, device=dev)
    x = wide[:, :1024].contiguous()
    assert torch.equal(apply_int8_linear(x, w.t(), one, sums), apply_int8_linear(x, w.t(), one.expand(64).contiguous(), sums))
    for asym in (None, sums):
        assert apply_int8_linear(x[:0], w.t(), sb, asym).shape == (0, 64)


def test_refusals(dev):
    from sglang_amd import int8_scaled_mm_azp
    from sglang_amd.quantization.int8_utils import apply_int8_linear, int8_weight_sums

    a, w, zp, sa, sb, bias = _operands(dev, 4, 64, 256, 1)
    sums = int8_weight_sums(w.t())
    good = dict(mat_a=a, mat_b=w.t(), scales_a=sa, scales_b=sb, out_dtype=torch.bfloat16, azp=zp, weight_sums=sums)
    int8_scaled_mm_azp(**good)
    for bad in (dict(mat_a=a.float()), dict(mat_b=w), dict(scales_a=sa[:3]), dict(scales_b=sb.double()), dict(out_dtype=torch.float32),
                dict(azp=zp.float()), dict(azp=zp[:2]), dict(weight_sums=sums[:8]), dict(weight_sums=sums.cpu()), dict(weight_sums=sums.long()),
                dict(bias=bias), dict(mat_a=a[:, :128])):
        with pytest.raises(RuntimeError):
            int8_scaled_mm_azp(**{**good, **bad})
    x = torch.zeros(4, 256, device=dev, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        apply_int8_linear(x, w.t(), sb, input_scale=sa)
    with pytest.raises(NotImplementedError):
        apply_int8_linear(x, w.t(), sb, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        apply_int8_linear(a, w.t(), sb)
    with pytest.raises(ValueError):
        apply_int8_linear(a, w.t(), sb, input_scale=sa, input_zero_point=zp)
    with pytest.raises(RuntimeError):
        apply_int8_linear(x.float(), w.t(), sb)
    with pytest.raises(NotImplementedError):
        apply_int8_linear(x.requires_grad_(), w.t(), sb)


@pytest.mark.parametrize("m,n,k", [(1, 512, 1024), (5, 520, 2048), (40, 8192, 4096), (300, 512, 8192), (300, 1024, 336)])
@pytest.mark.parametrize("asym", [False, True])
def test_linear_captured_and_replayed(dev, m, n, k, asym):
    """Rows quantised in the product, by a launch in front, K in slices: captured once, replayed on changing rows between eager calls."""
    from sglang_amd.quantization.int8_utils import apply_int8_linear, int8_weight_sums

    _, w, _, _, sb, bias = _operands(dev, 1, n, k, m)
    sums, bias = int8_weight_sums(w.t()) if asym else None, bias.bfloat16()
    g = torch.Generator().manual_seed(m)
    inputs = [torch.randn(m, k, generator=g).to(torch.bfloat16).to(dev) for _ in range(3)]
    x = inputs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        apply_int8_linear(x, w.t(), sb, sums, bias=bias)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = apply_int8_linear(x, w.t(), sb, sums, bias=bias)
    for i in range(6):
        want = apply_int8_linear(inputs[i % 3], w.t(), sb, sums, bias=bias)
        x.copy_(inputs[i % 3])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
