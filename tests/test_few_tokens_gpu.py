"""The expert layer of a few tokens on 8-bit rows against its definition in 64 bits, and the row-scaled operators in a row."""
import pytest
import torch

from . import row_layers as rl

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _layer(dev, m, e, topk, h, i, int8, seed, bias=None, ids=None):
    g = torch.Generator().manual_seed(seed)

    def codes(*shape):
        if int8:
            return torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)
        return (torch.randn(*shape, generator=g) * 100).clamp(-448, 448).to(F8)

    peak = 1.0 if int8 else 1.3
    t = dict(hidden_q=codes(m, h), hidden_scale=torch.rand(m, 1, generator=g) * 0.02 + 0.01, w1=codes(e, 2 * i, h), w2=codes(e, h, i),
             w1_scale=(torch.rand(e, 2 * i, 1, generator=g) + 0.5) * (2e-2 * peak / h ** 0.5), w2_scale=(torch.rand(e, h, 1, generator=g) + 0.5) * (1e-2 / i ** 0.5),
             topk_weights=torch.rand(m, topk, generator=g), topk_ids=ids if ids is not None else
             torch.stack([torch.randperm(e, generator=g)[:topk] if topk <= e else torch.randint(0, e, (topk,), generator=g) for _ in range(m)]).to(torch.int32))
    if bias is not None:
        t.update(b1=torch.randn(e, 2 * i, generator=g).to(bias), b2=torch.randn(e, h, generator=g).to(bias))
    return {k: v.to(dev) for k, v in t.items()}


def _check(out, t, factor=1.0):
    c = {k: v.cpu() for k, v in t.items()}
    want, off = rl.experts(c["hidden_q"], c["hidden_scale"], c["w1"], c["w2"], c["w1_scale"], c["w2_scale"], c["topk_weights"], c["topk_ids"],
                           c.get("b1"), c.get("b2"), factor)
    rl.check_rounded(out, want, rl.U, off)


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("m,e,topk,h,i", [
    (1, 8, 2, 256, 128), (1, 64, 6, 512, 256), (1, 1, 1, 16, 16), (2, 16, 4, 1024, 384), (3, 128, 8, 2048, 768), (4, 4, 4, 512, 640),
    (1, 4, 2, 7168, 2048), (2, 3, 3, 144, 2064), (5, 8, 3, 272, 48), (8, 32, 8, 640, 176), (64, 8, 1, 128, 64), (1, 70, 64, 128, 32),
    (4, 2, 2, 128, 4096), (2, 2, 1, 64, 16384), (7, 5, 5, 1040, 528), (16, 1, 1, 256, 512),
])
def test_layer(dev, int8, m, e, topk, h, i):
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens, takes_few_tokens

    assert takes_few_tokens(m, topk)
    t = _layer(dev, m, e, topk, h, i, int8, m + e + h)
    print(f"few tokens {m} x {topk} of {e}, {h} x {i}, int8 {int8}", flush=True)
    out = fused_experts_few_tokens(**t)
    _check(out, t)
    assert torch.equal(out, fused_experts_few_tokens(**t))


def test_intermediate_rows_whose_scale_has_no_reciprocal(dev):
    """Values of some 1e-38 and zeros between the products: 256 terms of at most 448 * 1e-36, and nothing that is not finite."""
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens

    t = _layer(dev, 2, 4, 2, 512, 256, False, 3)
    t["w1"].view(torch.int8)[:, 256 + 5] = 0
    t["w1_scale"][:, 256:] = 1e-40
    t["w2_scale"][:] = 1.0
    out = fused_experts_few_tokens(**t).cpu()
    assert torch.isfinite(out).all() and (out.abs() <= 2 * 256 * 448 * 1e-36).all()


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_biases_factor_and_types(dev, int8, dtype):
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens

    t = _layer(dev, 3, 16, 4, 512, 256, int8, 11, bias=dtype)
    _check(fused_experts_few_tokens(**t, out_dtype=dtype, routed_scaling_factor=2.5), t, 2.5)
    long = {**t, "topk_ids": t["topk_ids"].long(), "topk_weights": t["topk_weights"].to(torch.bfloat16).float()}
    _check(fused_experts_few_tokens(**long, out_dtype=dtype), long)
    # a token's row depends on its own experts only, whoever shares them
    every = fused_experts_few_tokens(**t, out_dtype=dtype)
    for k in range(3):
        alone = {**t, **{n: t[n][k:k + 1] for n in ("hidden_q", "hidden_scale", "topk_weights", "topk_ids")}}
        _check(fused_experts_few_tokens(**alone, out_dtype=dtype), alone)
        if int8:  # (whole sums are exact, so nothing depends on how many lanes share them)
            assert torch.equal(every[k:k + 1], fused_experts_few_tokens(**alone, out_dtype=dtype))


@pytest.mark.parametrize("int8", [True, False])
def test_ids_repeated_shared_and_elsewhere(dev, int8):
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens

    rows = [[[0] * 8] * 8, [[-1, 3, 3, 3, 99, 2, 2, -5]] * 5 + [[7, 6, 5, 4, 3, 2, 1, 0]] * 3, [[-1] * 8, [0, 1, 2, 3, 4, 5, 6, 7]],
            [[8] * 8], [[1, 1, 1, 1, 1, 1, 1, 0]] * 7]
    for n, ids in enumerate(rows):
        for dtype in (torch.int32, torch.int64):
            t = _layer(dev, len(ids), 8, 8, 256, 192, int8, n, ids=torch.tensor(ids, dtype=dtype))
            out = fused_experts_few_tokens(**t)
            _check(out, t)
            if all(not 0 <= i < 8 for i in ids[0]):
                assert not out[0].any()
    # an id of 64 bits whose low half names an expert is elsewhere too
    t = _layer(dev, 1, 8, 2, 256, 192, int8, 3, ids=torch.tensor([[3 + (1 << 32), 5]]))
    _check(fused_experts_few_tokens(**t), t)


def test_rows_and_values_that_are_zero_or_not_finite(dev):
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens

    for int8 in (True, False):
        t = _layer(dev, 4, 8, 2, 256, 128, int8, 21, ids=torch.tensor([[0, 1], [2, 3], [4, 5], [0, 4]], dtype=torch.int32))
        t["hidden_q"][1] = torch.zeros(256, dtype=t["hidden_q"].dtype)
        t["hidden_scale"][2] = float("nan")  # what a norm says of a row with a NaN
        out = fused_experts_few_tokens(**t)
        assert not out[1].any() and out[2].isnan().all() and torch.isfinite(out[[0, 3]]).all()
        c = {k: (v[[0, 1, 3]] if v.shape[0] == 4 else v) for k, v in t.items()}
        _check(out[[0, 1, 3]], c)


def test_no_tokens_and_refusals(dev):
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens, takes_few_tokens

    t = _layer(dev, 2, 8, 2, 256, 128, True, 1)
    none = {**t, **{n: t[n][:0] for n in ("hidden_q", "hidden_scale", "topk_weights", "topk_ids")}}
    assert fused_experts_few_tokens(**none).shape == (0, 256)
    many = _layer(dev, 13, 8, 5, 256, 128, True, 1)
    assert not takes_few_tokens(13, 5)
    with pytest.raises(NotImplementedError):
        fused_experts_few_tokens(**many)
    for bad in (dict(hidden_q=t["hidden_q"].float()), dict(hidden_q=t["hidden_q"][:, :128]), dict(w1=t["w1"].view(torch.uint8)), dict(w1=t["w1"][:, ::2]),
                dict(w2=t["w2"][:4]), dict(hidden_scale=t["hidden_scale"][:1]), dict(w1_scale=t["w1_scale"][:, :128]), dict(w2_scale=t["w2_scale"].half()),
                dict(topk_ids=t["topk_ids"].float()), dict(topk_ids=t["topk_ids"][:, :1]), dict(out_dtype=torch.float32), dict(topk_ids=t["topk_ids"].cpu()),
                dict(b1=torch.zeros(8, 256, device=dev))):
        with pytest.raises(RuntimeError):
            fused_experts_few_tokens(**{**t, **bad})
    with pytest.raises(RuntimeError):
        fused_experts_few_tokens(**_layer(dev, 1, 2, 1, 24, 16, True, 1))  # H no multiple of 16


def _block(dev, dtype=torch.bfloat16, rows=5, h=512, i=640, e=16, topk=2):
    """A decoder block's row-scaled parts: norm -> int8 linear, norm -> experts, SiLU -> int8 linear."""
    g = torch.Generator().manual_seed(77)
    w = torch.randint(-127, 128, (2 * i, h), generator=g, dtype=torch.int8).to(dev)
    w_down = torch.randint(-127, 128, (h, i), generator=g, dtype=torch.int8).to(dev)
    p = dict(gamma=(torch.rand(h, generator=g) + 0.5).to(dtype).to(dev), w=w, sw=(torch.rand(2 * i, 1, generator=g) * 1e-3).to(dev), w_down=w_down,
             sd=(torch.rand(h, 1, generator=g) * 1e-3).to(dev))
    p.update({k: v for k, v in _layer(dev, rows, e, topk, h, 256, True, 5).items() if not k.startswith("hidden")})
    return p


def _run_block(p, x, res):
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant, silu_and_mul_row_quant
    from sglang_amd.quantization.int8_utils import apply_int8_linear

    (q, s, zp), _, res1 = fused_rms_row_quant(x, p["gamma"], 1e-6, res=res, symmetric=False)
    mid = apply_int8_linear(q, p["w"].t(), p["sw"], weight_sums=p["sums"], input_scale=s, input_zero_point=zp, out_dtype=x.dtype)
    q2, s2, zp2 = silu_and_mul_row_quant(mid, symmetric=False)
    out = apply_int8_linear(q2, p["w_down"].t(), p["sd"], weight_sums=p["sums_down"], input_scale=s2, input_zero_point=zp2, out_dtype=x.dtype)
    (q3, s3), y, res2 = fused_rms_row_quant(out, p["gamma"], 1e-6, res=res1, output_unquantized=True)
    moe = fused_experts_few_tokens(q3, s3, p["w1"], p["w2"], p["w1_scale"], p["w2_scale"], p["topk_weights"], p["topk_ids"], out_dtype=x.dtype)
    return out, y, res2, moe


def _with_sums(p):
    from sglang_amd.quantization.int8_utils import int8_weight_sums

    return dict(p, sums=int8_weight_sums(p["w"].t()), sums_down=int8_weight_sums(p["w_down"].t()))


def test_a_block_of_them(dev):
    """Each operator on the outputs of the one in front, each held to its own definition."""
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant, silu_and_mul_row_quant
    from sglang_amd.quantization.int8_utils import apply_int8_linear

    p = _with_sums(_block(dev))
    g = torch.Generator().manual_seed(8)
    x, res = (torch.randn(5, 512, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    (q, s, zp), _, res1 = fused_rms_row_quant(x, p["gamma"], 1e-6, res=res, symmetric=False)
    v64, y64 = rl.rms(x.cpu(), p["gamma"].cpu(), 1e-6, res.cpu())
    rl.check_codes(y64, rl.rms_error(512), q, s, zp)
    mid = apply_int8_linear(q, p["w"].t(), p["sw"], weight_sums=p["sums"], input_scale=s, input_zero_point=zp)
    rl.check_product(mid, q, zp, p["w"], s, p["sw"], None)
    q2, s2, zp2 = silu_and_mul_row_quant(mid, symmetric=False)
    rl.check_codes(rl.silu_mul(mid.cpu()), rl.silu_error(mid.cpu()), q2, s2, zp2)
    out = apply_int8_linear(q2, p["w_down"].t(), p["sd"], weight_sums=p["sums_down"], input_scale=s2, input_zero_point=zp2)
    rl.check_product(out, q2, zp2, p["w_down"], s2, p["sd"], None)
    (q3, s3), y, res2 = fused_rms_row_quant(out, p["gamma"], 1e-6, res=res1, output_unquantized=True)
    t = dict({k: p[k] for k in ("w1", "w2", "w1_scale", "w2_scale", "topk_weights", "topk_ids")}, hidden_q=q3, hidden_scale=s3)
    moe = fused_experts_few_tokens(**t)
    _check(moe, t)
    assert all(torch.equal(a, b) for a, b in zip((out, y, res2, moe), _run_block(p, x, res)))


@pytest.mark.parametrize("static", [False, True])
def test_an_fp8_block_of_them(dev, static):
    """Norm -> fp8_scaled_mm -> SiLU -> fp8_scaled_mm -> norm -> e4m3 experts, per token and with given scales."""
    from sglang_amd import fp8_scaled_mm
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant, silu_and_mul_row_quant

    g = torch.Generator().manual_seed(3)
    x, res = (torch.randn(6, 512, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    gamma = (torch.rand(512, generator=g) + 0.5).to(dev)
    w_up, w_down = ((torch.randn(*s, generator=g) * 100).clamp(-448, 448).to(F8).to(dev) for s in ((1280, 512), (512, 640)))
    s_up, s_down = torch.full((1280, 1), 2e-4, device=dev), torch.full((512, 1), 2e-4, device=dev)
    given = [torch.full((1,), v, device=dev) if static else None for v in (0.01, 0.004, 0.01)]

    def fixed(scale):
        return None if scale is None else float(scale)

    def product(q, s, w, ws):
        out = fp8_scaled_mm(q, w.t(), s, ws, torch.bfloat16)
        a, b = q.cpu().float().double(), w.cpu().float().double()
        scale = s.cpu().double() * ws.cpu().double().view(1, -1)
        # 512 to 640 products, summed in 32 bits, times two scales
        rl.check_rounded(out, (a @ b.t()) * scale, 3 * rl.U, (a.abs() @ b.abs().t()) * scale * 640 * rl.U)
        return out

    (q, s), _, r1 = fused_rms_row_quant(x, gamma, 1e-6, res=res, dtype_quant=F8, scale=given[0])
    rl.check_codes(rl.rms(x.cpu(), gamma.cpu(), 1e-6, res.cpu())[1], rl.rms_error(512), q, s, None, fixed(given[0]))
    mid = product(q, s, w_up, s_up)
    q, s = silu_and_mul_row_quant(mid, dtype_quant=F8, scale=given[1])
    rl.check_codes(rl.silu_mul(mid.cpu()), rl.silu_error(mid.cpu()), q, s, None, fixed(given[1]))
    out = product(q, s, w_down, s_down)
    (q, s), y, _ = fused_rms_row_quant(out, gamma, 1e-6, res=r1, dtype_quant=F8, scale=given[2], output_unquantized=True)
    rl.check_rounded(y, rl.rms(out.cpu(), gamma.cpu(), 1e-6, r1.cpu())[1], rl.rms_error(512))
    t = dict({k: v for k, v in _layer(dev, 6, 16, 2, 512, 256, False, 8).items() if not k.startswith("hidden")}, hidden_q=q, hidden_scale=s)
    _check(fused_experts_few_tokens(**t), t)


def test_captured_and_replayed(dev):
    """The run captured into two graphs that share a pool, replayed in turn on changing inputs with eager work between."""
    p = _with_sums(_block(dev))
    g = torch.Generator().manual_seed(9)
    inputs = [tuple(torch.randn(5, 512, generator=g).to(torch.bfloat16).to(dev) for _ in range(2)) for _ in range(4)]
    x, res = (t.clone() for t in inputs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run_block(p, x, res)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(_run_block(p, x, res))
        graphs.append(graph)
    for n in range(6):
        a, b = inputs[n % 4]
        want = _run_block(p, a, b)
        x.copy_(a)
        res.copy_(b)
        graphs[n % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(outs[n % 2], want)), n


def test_on_two_streams_at_once(dev):
    p = _with_sums(_block(dev))
    g = torch.Generator().manual_seed(10)
    inputs = [tuple(torch.randn(5, 512, generator=g).to(torch.bfloat16).to(dev) for _ in range(2)) for _ in range(2)]
    want = [_run_block(p, *i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    got = []
    for _ in range(20):
        for s, i in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append(_run_block(p, *i))
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for n, o in enumerate(got) for u, v in zip(o, want[n % 2]))


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("m,e,topk,h,i", [(3, 40, 8, 2048, 768), (1, 80, 64, 1024, 1024), (9, 6, 1, 528, 1024), (6, 3, 10, 80, 16), (5, 64, 2, 4064, 1008)])
def test_more_pairs_than_eight_waves_take_at_once(dev, int8, m, e, topk, h, i):
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens

    t = _layer(dev, m, e, topk, h, i, int8, m * e + i, bias=torch.bfloat16)
    print(f"few tokens {m} x {topk} of {e}, {h} x {i}, int8 {int8}", flush=True)
    _check(fused_experts_few_tokens(**t), t)
