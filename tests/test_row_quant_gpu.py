"""RMSNorm (+ residual), SiLU * up and plain rows to 8-bit codes with one scale per row, against the definitions in 64 bits."""
import pytest
import torch

from . import row_layers as rl

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
KINDS = ["fp8", "static", "int8", "asym"]
FIXED = 0.011


def _options(kind, dev):
    return dict(dtype_quant=F8 if kind in ("fp8", "static") else torch.int8, symmetric=kind != "asym",
                scale=torch.full((1,), FIXED, device=dev) if kind == "static" else None)


def _check(y, error, codes, kind):
    rl.check_codes(y, error, codes[0], codes[1], codes[2] if kind == "asym" else None, float(torch.tensor(FIXED)) if kind == "static" else None)


def _rows(g, *shape, dtype=torch.bfloat16, shift=0.0):
    return (torch.randn(*shape, generator=g) * 2 + shift).to(dtype)


# (teams of a wave, one workgroup form after the other, each with pieces that are aligned and with pieces that overlap at the end, the
# value-by-value form: fewer than 8 values and more than 32768)
ROW_SIZES = [(1, 1), (3, 7), (2, 8), (5, 24), (1, 128), (700, 512), (600, 1000), (40, 1000), (600, 2000), (37, 1536), (1, 7168), (530, 4096), (515, 8192),
             (7, 8184), (9, 16384), (3, 28672), (2, 32776), (4, 4099), (3, 9), (5, 15), (700, 513), (600, 1001), (40, 1023), (600, 2046), (37, 1537), (530, 4095),
             (515, 8191), (9, 16383), (3, 28673), (2, 32767)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,hidden", ROW_SIZES)
@pytest.mark.parametrize("dtype,wtype,residual", [(torch.bfloat16, torch.bfloat16, True), (torch.float16, torch.float32, True),
                                                  (torch.bfloat16, torch.float32, False), (torch.float16, torch.float16, False)])
def test_norm(dev, kind, rows, hidden, dtype, wtype, residual):
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant

    g = torch.Generator().manual_seed(rows * 1000 + hidden)
    x, res = _rows(g, rows, hidden, dtype=dtype), _rows(g, rows, hidden, dtype=dtype) if residual else None
    w = (torch.rand(hidden, generator=g) + 0.5).to(wtype)
    codes, y, res_out = fused_rms_row_quant(x.to(dev), w.to(dev), 1e-6, res=None if res is None else res.to(dev), output_unquantized=rows % 2 == 1,
                                            **_options(kind, dev))
    v64, y64 = rl.rms(x, w, 1e-6, res)
    _check(y64, rl.rms_error(hidden), codes, kind)
    assert (res_out is not None) == residual and (y is not None) == (rows % 2 == 1)
    if residual:
        assert torch.equal(res_out.cpu(), (x.float() + res.float()).to(dtype))
    if y is not None:
        rl.check_rounded(y, y64, rl.rms_error(hidden))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,hidden", ROW_SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_silu(dev, kind, rows, hidden, dtype):
    from sglang_amd.quantization.fused_row_quant import silu_and_mul_row_quant

    g = torch.Generator().manual_seed(rows * 1000 + hidden)
    x = _rows(g, rows, 2 * hidden, dtype=dtype, shift=0.3)
    _check(rl.silu_mul(x), rl.silu_error(x), silu_and_mul_row_quant(x.to(dev), **_options(kind, dev)), kind)


@pytest.mark.parametrize("rows,hidden", ROW_SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_zero_points_of_plain_rows(dev, rows, hidden, dtype):
    from sglang_amd.quantization.int8_kernel import per_token_quant_int8_asym

    g = torch.Generator().manual_seed(rows * 1000 + hidden)
    x = _rows(g, rows, hidden, dtype=dtype, shift=rows % 3 * 1.5 - 1.5)  # rows on either side of zero, and across it
    _check(x.double(), 0.0, per_token_quant_int8_asym(x.to(dev)), "asym")
    q, s, zp = per_token_quant_int8_asym(x.to(dev).view(rows, 1, hidden))
    assert q.shape == (rows, 1, hidden) and s.shape == zp.shape == (rows, 1, 1)


@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_zeros_and_rows_that_a_few_values_fill(dev, kind):
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant, silu_and_mul_row_quant

    x = torch.zeros(6, 256, dtype=torch.bfloat16)
    x[1, 17] = 3e4  # one value
    x[2] = -0.0
    x[3] = 1e-30  # squares that vanish
    x[4, ::2], x[4, 1::2] = 2.0, -2.0
    x[5, 255] = -1e-3
    w = torch.ones(256)
    codes, y, _ = fused_rms_row_quant(x.to(dev), w.to(dev), 1e-6, output_unquantized=True, **_options(kind, dev))
    _, y64 = rl.rms(x, w, 1e-6)
    _check(y64, rl.rms_error(256), codes, kind)
    xx = torch.cat([x, x.flip(0)], dim=1)
    _check(rl.silu_mul(xx), rl.silu_error(xx), silu_and_mul_row_quant(xx.to(dev), **_options(kind, dev)), kind)


@pytest.mark.parametrize("hidden", [64, 1024, 8192, 333])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_with_a_nan_or_an_infinity_stay_visible(dev, hidden, bad):
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant, silu_and_mul_row_quant
    from sglang_amd.quantization.int8_kernel import per_token_quant_int8_asym

    g = torch.Generator().manual_seed(hidden)
    x = _rows(g, 4, hidden)
    x[2, hidden // 2 + 1] = bad
    xx = torch.cat([x, _rows(g, 4, hidden)], dim=1)
    w = torch.ones(hidden)
    for kind in KINDS:
        outs = [fused_rms_row_quant(x.to(dev), w.to(dev), 1e-6, **_options(kind, dev))[0], silu_and_mul_row_quant(xx.to(dev), **_options(kind, dev))]
        if kind == "asym":
            outs.append(per_token_quant_int8_asym(x.to(dev)))
        for codes in outs:
            finite = torch.isfinite(codes[1].cpu()).view(-1)
            if kind == "static":
                # (an infinity behind the SiLU is clamped to the largest code, as any value beyond the given scale)
                spoilt = codes[0].cpu().float().isnan().any(dim=1) | (codes[0].cpu().float().abs() == 448).any(dim=1) | (bad == float("-inf"))
                assert finite.all() and spoilt[2] and not codes[0].cpu().float().isnan()[[0, 1, 3]].any()
            else:
                assert finite.tolist() == [True, True, False, True], kind


@pytest.mark.parametrize("hidden", [64, 1024, 8192, 333])
@pytest.mark.parametrize("weight,value", [(float("nan"), 1.0), (float("inf"), 1.0), (float("inf"), 0.0)])
def test_a_norm_with_a_bad_weight_stays_visible(dev, hidden, weight, value):
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant

    x = _rows(torch.Generator().manual_seed(hidden), 3, hidden)
    w = torch.ones(hidden)
    w[hidden // 2 + 1], x[:, hidden // 2 + 1] = weight, value
    for kind in ("fp8", "int8", "asym"):
        assert not torch.isfinite(fused_rms_row_quant(x.to(dev), w.to(dev), 1e-6, **_options(kind, dev))[0][1]).any(), kind


@pytest.mark.parametrize("hidden", [64, 1024, 8192, 333])
def test_values_whose_scale_has_no_reciprocal(dev, hidden):
    """Zeros stay zeros, and what is lost is below 1e-36 times what the norm multiplies by (1 / sqrt(eps))."""
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant, silu_and_mul_row_quant

    x = torch.zeros(2, hidden, dtype=torch.bfloat16)
    x[0, ::3], x[1, 5], x[1, 7] = 1e-38, -3e-38, 1e-36
    up = torch.cat([torch.full_like(x, 4.0), x], dim=1)
    (q, s), _, _ = fused_rms_row_quant(x.to(dev), torch.ones(hidden, device=dev), 1e-6, dtype_quant=F8)
    qs, ss = silu_and_mul_row_quant(up.to(dev), dtype_quant=F8)
    for codes, scale, y, lost in ((q, s, rl.rms(x, torch.ones(hidden), 1e-6)[1], 2e-33), (qs, ss, rl.silu_mul(up), 1e-35)):
        c = codes.cpu().float()
        assert (c[x == 0] == 0).all()
        assert ((c.double() * scale.cpu().double() - y).abs() <= lost).all()


@pytest.mark.parametrize("rows,hidden", [((1 << 22) + 3, 8), ((1 << 20) + 1, 1032), ((1 << 24) + 5, 3)])
def test_more_rows_than_one_grid_dimension_holds(dev, rows, hidden):
    from sglang_amd.quantization.int8_kernel import per_token_quant_int8_asym

    g = torch.Generator().manual_seed(hidden)
    some = _rows(g, 1009, hidden, dtype=torch.float16, shift=0.5).to(dev)
    x = some.repeat(rows // 1009 + 1, 1)[:rows]
    want = per_token_quant_int8_asym(some)
    for got, part in zip(per_token_quant_int8_asym(x), want):
        assert got.shape[0] == rows
        whole = rows // 1009 * 1009
        assert (got[:whole].view(-1, 1009, got.shape[1]) == part).all() and torch.equal(got[whole:], part[:rows - whole])


def test_the_other_rows_do_not_see_a_bad_one(dev):
    from sglang_amd.quantization.fused_row_quant import silu_and_mul_row_quant

    g = torch.Generator().manual_seed(5)
    x = _rows(g, 2048, 256).to(dev)
    good = silu_and_mul_row_quant(x)
    x[1::2] = float("nan")
    both = silu_and_mul_row_quant(x)
    assert torch.equal(good[0][::2], both[0][::2]) and torch.equal(good[1][::2], both[1][::2])


def test_views_strides_alignment(dev):
    """Columns of a wider tensor, rows that start off 16 bytes, one row repeated: the same bits as the copies of them."""
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant, silu_and_mul_row_quant
    from sglang_amd.quantization.int8_kernel import per_token_quant_int8_asym

    g = torch.Generator().manual_seed(6)
    wide = _rows(g, 9, 4096).to(dev)
    w = torch.rand(1024, generator=g).to(dev)
    views = [wide[:, 512:1536], wide[::3, :1024], wide[:1, 8:1032], wide[2:3, :1024].expand(5, 1024), wide[:, 1:1025], wide[::2, 1003:2027]]
    for i, v in enumerate(views):
        copy = v.contiguous()
        for kind in KINDS:
            o = _options(kind, dev)
            a, ya, ra = fused_rms_row_quant(v, w, 1e-5, res=v, output_unquantized=True, **o)
            b, yb, rb = fused_rms_row_quant(copy, w, 1e-5, res=copy, output_unquantized=True, **o)
            assert torch.equal(ra, rb)
            # (values one by one add up in another order)
            y64 = rl.rms(copy.cpu(), w.cpu(), 1e-5, copy.cpu())[1]
            for out, y in ((a, ya), (b, yb)):
                _check(y64, rl.rms_error(1024), out, kind)
                rl.check_rounded(y, y64, rl.rms_error(1024))
            if i < 4:
                assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a, b)) and torch.equal(ya, yb)
            s = silu_and_mul_row_quant(v, **o)
            assert all(torch.equal(p.contiguous().view(torch.uint8), q.contiguous().view(torch.uint8)) for p, q in zip(s, silu_and_mul_row_quant(copy, **o)))
        assert all(torch.equal(p, q) for p, q in zip(per_token_quant_int8_asym(v), per_token_quant_int8_asym(copy)))


def test_no_rows(dev):
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant, silu_and_mul_row_quant
    from sglang_amd.quantization.int8_kernel import per_token_quant_int8_asym

    x = torch.empty(0, 256, device=dev, dtype=torch.bfloat16)
    (q, s), y, r = fused_rms_row_quant(x, torch.ones(256, device=dev), 1e-6, res=x, output_unquantized=True)
    assert q.shape == (0, 256) and s.shape == (0, 1) and y.shape == r.shape == (0, 256)
    assert [t.shape[0] for t in silu_and_mul_row_quant(x, symmetric=False)] == [0, 0, 0]
    assert [t.shape[0] for t in per_token_quant_int8_asym(x)] == [0, 0, 0]


def test_refusals(dev):
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant, silu_and_mul_row_quant
    from sglang_amd.quantization.int8_kernel import per_token_quant_int8_asym
    from sglang_amd.quantization.int8_utils import int8_weight_sums

    x, w = torch.zeros(4, 64, device=dev, dtype=torch.bfloat16), torch.ones(64, device=dev)
    one = torch.ones(1, device=dev)
    for bad in (dict(inp=x.float()), dict(inp=x[0]), dict(inp=x.t()), dict(weight=w[:32]), dict(weight=w.half()), dict(weight=w.cpu()),
                dict(res=x[:2]), dict(res=x.half()), dict(dtype_quant=torch.uint8), dict(dtype_quant=F8, symmetric=False), dict(scale=one),
                dict(dtype_quant=F8, scale=torch.ones(2, device=dev)), dict(dtype_quant=F8, scale=one.half()), dict(dtype_quant=F8, scale=one.cpu())):
        with pytest.raises(RuntimeError):
            fused_rms_row_quant(**{**dict(inp=x, weight=w, epsilon=1e-6), **bad})
    for bad in (x.float(), x[:, :63], x[0], x.cpu()):
        with pytest.raises(RuntimeError):
            silu_and_mul_row_quant(bad)
    with pytest.raises(RuntimeError):
        per_token_quant_int8_asym(x.to(torch.int32))
    with pytest.raises(RuntimeError):
        int8_weight_sums(torch.zeros(8, 64, device=dev, dtype=torch.int8))  # rows, not the column-major view
    needs_grad = x.clone().requires_grad_()
    with pytest.raises(NotImplementedError):
        silu_and_mul_row_quant(needs_grad)
    with torch.no_grad():
        silu_and_mul_row_quant(needs_grad)
    with pytest.raises(NotImplementedError):
        torch.vmap(lambda row: per_token_quant_int8_asym(row)[0])(x.view(2, 2, 64))


@pytest.mark.parametrize("n,k", [(1, 1), (5, 16), (300, 4096), (7, 33), (64, 70000)])
def test_weight_sums(dev, n, k):
    from sglang_amd.quantization.int8_utils import int8_weight_sums

    g = torch.Generator().manual_seed(n + k)
    w = torch.randint(-128, 128, (n, k + 3), generator=g, dtype=torch.int8)
    assert torch.equal(int8_weight_sums(w[:, :k].contiguous().to(dev).t()).cpu(), w[:, :k].sum(dim=1, dtype=torch.int32))
    assert torch.equal(int8_weight_sums(w.to(dev)[:, 1:k + 1].t()).cpu(), w[:, 1:k + 1].sum(dim=1, dtype=torch.int32))
