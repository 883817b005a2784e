"""Arguments that the row-scaled operators refuse before any launch, through the C ABI and the Python functions; and the plain
model of them against small numbers worked by hand."""
import pytest
import torch

from . import row_layers as rl


def _lib():
    from sglang_amd._lib import lib

    return lib


def test_rms_row_quant_refuses():
    f = _lib().sglamd_fused_rms_row_quant
    # x, x_stride, res, res_stride, w, eps, fixed, rows, hidden, q, s, zp, y, res_out, dtype, weight_dtype, q_dtype, stream
    good = [64, 128, None, 0, 64, 1e-6, None, 4, 128, 64, 64, None, None, None, 2, 2, 4, None]
    for at, value, code in ((0, None, -1), (4, None, -1), (9, None, -1), (10, None, -1), (1, 64, -1), (1, -8, -1), (7, -1, -1), (7, 1 << 31, -1),
                            (8, 0, -1), (14, 0, -1), (15, 1, -1), (16, 5, -1), (2, 64, -1), (13, 64, -1), (6, 64, -2)):
        args = list(good)
        args[at] = value
        assert f(*args) == code, (at, value, _lib().sglamd_last_error())
    assert f(*[0 if i == 7 else v for i, v in enumerate(good)]) == 0  # no rows: nothing to do
    zp_with_fp8 = [64 if i == 11 else 3 if i == 16 else v for i, v in enumerate(good)]
    assert f(*zp_with_fp8) == -1
    short_res = [64 if i in (2, 13) else 64 if i == 3 else v for i, v in enumerate(good)]
    assert f(*short_res) == -1 and b"residual" in _lib().sglamd_last_error()


def test_silu_and_plain_rows_refuse():
    f = _lib().sglamd_silu_mul_row_quant
    good = [64, 256, None, 4, 128, 64, 64, None, 2, 4, None]
    for at, value in ((0, None), (1, 128), (3, -1), (4, 0), (5, None), (6, None), (8, 0), (8, 3), (9, 2)):
        args = list(good)
        args[at] = value
        assert f(*args) == -1, (at, value)
    assert f(*[64 if i == 2 else v for i, v in enumerate(good)]) == -2  # a given scale with int8 codes
    assert f(*[0 if i == 3 else v for i, v in enumerate(good)]) == 0
    f = _lib().sglamd_per_token_quant_int8_asym
    good = [64, 128, 2, 4, 128, 64, 64, 64, None]
    for at, value in ((0, None), (1, 100), (2, 3), (3, -1), (4, 0), (5, None), (6, None), (7, None)):
        args = list(good)
        args[at] = value
        assert f(*args) == -1, (at, value)
    f = _lib().sglamd_int8_weight_sums
    for args in ((None, 64, 4, 64, 64, None), (64, 32, 4, 64, 64, None), (64, 64, 4, 0, 64, None), (64, 64, 4, 64, None, None),
                 (64, 1 << 25, 4, 1 << 24, 64, None), (64, 64, -1, 64, 64, None)):
        assert f(*args) == -1, args


def test_asymmetric_product_refuses():
    f = _lib().sglamd_int8_scaled_mm_azp
    # a, lda, b, ldb, sa, sb, zp, sums, bias, out, ldc, dtype, M, N, K, ws, ws_bytes, stream
    good = [64, 256, 64, 256, 64, 64, 64, 64, None, 64, 64, 2, 4, 64, 256, None, 0, None]
    for at, value, code in ((0, None, -1), (2, None, -1), (4, None, -1), (5, None, -1), (6, None, -1), (7, None, -1), (9, None, -1), (1, 128, -1),
                            (14, 248, -1), (14, 65552, -2), (0, 68, -1), (10, 32, -1)):
        args = list(good)
        args[at] = value
        if at == 14 and value > 256:
            args[1] = args[3] = value
        assert f(*args) == code, (at, value, _lib().sglamd_last_error())
    assert f(*[0 if i == 12 else v for i, v in enumerate(good)]) == 0


def test_int8_linear_refuses():
    f = _lib().sglamd_int8_row_linear
    # x, x_stride, dtype, M, K, w, ldb, sb, sums, bias, out, ldc, N, q, sa, zp, ws, ws_bytes, stream
    good = [64, 256, 2, 4, 256, 64, 256, 64, 64, None, 64, 64, 64, 64, 64, 64, None, 0, None]
    for at, value, code in ((0, None, -1), (5, None, -1), (7, None, -1), (10, None, -1), (13, None, -1), (14, None, -1), (15, None, -1), (2, 0, -1),
                            (1, 128, -1), (6, 128, -1), (11, 32, -1), (3, -1, -1), (12, 0, -1)):
        args = list(good)
        args[at] = value
        assert f(*args) == code, (at, value, _lib().sglamd_last_error())
    long = list(good)
    long[1] = long[4] = long[6] = 65552
    assert f(*long) == -2
    assert f(*[0 if i == 3 else v for i, v in enumerate(good)]) == 0


def test_few_tokens_refuses():
    f, w = _lib().sglamd_fused_experts_few_tokens, _lib().sglamd_fused_experts_few_tokens_workspace
    assert w(4, 256, 8) == 4 * 8 * 256 * 4 and w(0, 256, 8) == 0 and w(1 << 40, 1 << 40, 8) == 0
    # x, xs, q_dtype, M, H, I, E, topk, w13, s13, b13, w2, s2, b2, weights, ids, ids_dtype, out, out_dtype, factor, ws, bytes, stream
    good = [64, 64, 4, 2, 256, 128, 8, 2, 64, 64, None, 64, 64, None, 64, 64, 5, 64, 2, 1.0, 64, 1 << 20, None]
    for at, value, code in ((0, None, -1), (1, None, -1), (8, None, -1), (9, None, -1), (11, None, -1), (12, None, -1), (14, None, -1), (15, None, -1),
                            (17, None, -1), (20, None, -1), (2, 2, -1), (18, 0, -1), (16, 2, -1), (3, 0, -1), (6, 0, -1), (7, 0, -1), (3, 33, -2),
                            (7, 65, -2), (4, 264, -1), (5, 120, -1), (5, 16400, -2), (4, 32784, -2), (0, 72, -1), (20, 72, -1), (21, 1000, -1),
                            (4, 1 << 24, -2), (3, 1 << 40, -2)):
        args = list(good)
        args[at] = value
        assert f(*args) == code, (at, value, _lib().sglamd_last_error())


def test_functions_refuse_host_tensors():
    from sglang_amd import int8_scaled_mm_azp
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens, takes_few_tokens
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant, silu_and_mul_row_quant
    from sglang_amd.quantization.int8_kernel import per_token_quant_int8_asym
    from sglang_amd.quantization.int8_utils import apply_int8_linear, int8_weight_sums

    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(16, 64, dtype=torch.int8)
    i, s = torch.zeros(16, dtype=torch.int32), torch.ones(16)
    for call in (lambda: fused_rms_row_quant(x, torch.ones(64), 1e-6), lambda: silu_and_mul_row_quant(x), lambda: per_token_quant_int8_asym(x),
                 lambda: int8_weight_sums(w.t()), lambda: apply_int8_linear(x, w.t(), s), lambda: apply_int8_linear(x, w.t(), s, i),
                 lambda: int8_scaled_mm_azp(w[:4], w.t(), s[:4], s, torch.bfloat16, i[:4], i),
                 lambda: fused_experts_few_tokens(w, s, w.view(1, 16, 64), w.view(1, 64, 16)[:, :, :8], s, s, s.view(16, 1), i.view(16, 1))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    assert takes_few_tokens(8, 8) and not takes_few_tokens(13, 5)


def test_the_model_of_the_rows():
    y = torch.tensor([[0.0, 2.54, -1.27], [-1.0, -3.0, -2.55], [0.0, 0.0, 0.0]], dtype=torch.float64)
    assert torch.allclose(rl.symmetric(y, True).view(-1), torch.tensor([0.02, 3 / 127, 1e-10 / 127], dtype=torch.float64))
    scale, zp = rl.asymmetric(y)
    assert torch.allclose(scale.view(-1), torch.tensor([3.81 / 255, 3 / 255, 1e-10 / 255], dtype=torch.float64))
    assert torch.allclose(zp.view(-1), torch.tensor([-128 + 1.27 * 255 / 3.81, 127.0, -128.0], dtype=torch.float64))
    q = torch.tensor([[0, 127, -64], [-42, -127, -108], [0, 0, 0]], dtype=torch.int8)
    s = torch.tensor([[0.02], [3 / 127], [1e-10 / 127]])
    rl.check_codes(y, 0.0, q, s)
    with pytest.raises(AssertionError):
        rl.check_codes(y, 0.0, torch.where(q == 127, 126, q).to(torch.int8), s)  # a code that is one step off
    with pytest.raises(AssertionError):
        rl.check_codes(y, 0.0, q, s * 1.001)


def test_the_model_of_the_experts():
    x, w1 = torch.tensor([[1, 0]], dtype=torch.int8), torch.tensor([[[100, 3], [2, 5]]], dtype=torch.int8)
    w2 = torch.tensor([[[3], [-7]]], dtype=torch.int8)
    one = torch.ones(1, 2, 1)
    out, off = rl.experts(x, torch.ones(1, 1), w1, w2, one, one, torch.tensor([[0.5]]), torch.tensor([[0]]))
    # silu(100) * 2 = 200 is the row's largest: code 127 at a scale of 200 / 127
    assert torch.allclose(out, torch.tensor([[300.0, -700.0]], dtype=torch.float64)) and (off < out.abs() * 1e-5).all()
    assert not rl.experts(x, torch.ones(1, 1), w1, w2, one, one, torch.tensor([[0.5]]), torch.tensor([[-1]]))[0].any()
