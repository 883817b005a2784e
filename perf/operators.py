"""Operators of layers whose activations carry one scale per token ("row-scaled" layers), as cases that can be prepared,
run in a plain form or through this library, and priced.

  norm     residual addition and RMSNorm with an output in 8 bits: e4m3 codes and a scale per token (or one scale known
           beforehand), or int8 codes and a scale per token.  What stands in front of the first product of a block.
  silu     SiLU(gate) * up of a [gate | up] row with the same outputs.  What stands between the products of an MLP.
  linear   a linear layer on int8 weights with a scale per output channel and int8 activations with a scale AND a zero
           point per token (asymmetric).  Its rows come as 16-bit values ("rows"), or out of a norm ("norm") or a SiLU
           ("silu") that leaves int8 codes, scales and zero points.
  moe      the whole expert layer of a few tokens whose rows are in 8 bits already (a norm's codes and scales), experts with
           a scale per output channel, e4m3 or int8.

Definitions (x real, i.e. nothing is rounded unless it says so; round() is to nearest):

  norm     v = x + residual;  y = v / sqrt(mean(v^2) + eps) * gamma;  the updated residual is v in the layer's type
  silu     y = gate / (1 + exp(-gate)) * up
  e4m3     scale = max|y| / 448 (or as given);  code = e4m3(clamp(y / scale, -448, 448));  zeros where the scale is 0
  int8     amax = max(max|y|, 1e-10);  scale = amax / 127;  code = round(y / scale)
  asym     lo = min(0, min y), hi = max(0, max y);  scale = max(hi - lo, 1e-10) / 255;  zp = round(-128 - lo / scale);
           code = clamp(round(y / scale) + zp, -128, 127)
  linear   out[m, n] = scale[m] * wscale[n] * sum_k (code[m, k] - zp[m]) * w[n, k] + bias[n]
  moe      h = hscale[t] * w13scale[e] * (codes of token t times the expert's [gate | up] rows);  a = silu(gate) * up, in 8
           bits per (token, expert) row as above;  out[t] = sum over the token's experts of its routing weight times
           ascale * w2scale[e] * (codes of a times the expert's down rows)

Sizes are those of the benchmark's DeepSeek-V3 and Llama-3-70B layers, of the tests' layers, and generic ones."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
F8 = torch.float8_e4m3fn
EPS = 1e-6


def listed():
    return [
        # the layer input of one decoded token: residual, norm, codes for a per-token FP8 projection
        dict(name="norm_fp8_decode_1", path="norm", rows=1, hidden=7168, dtype="bf16", quant="fp8", residual=True, y=False, gamma="same"),
        # a small ragged decode batch on a short row, weights kept in 32 bits, the 16-bit row wanted too
        dict(name="norm_int8_decode_37", path="norm", rows=37, hidden=1536, dtype="f16", quant="int8", residual=False, y=True, gamma="f32"),
        # a prefill chunk
        dict(name="norm_fp8_prefill_4096", path="norm", rows=4096, hidden=8192, dtype="bf16", quant="fp8", residual=True, y=False, gamma="same"),
        # between the two products of an MLP: a few decoded tokens, a ragged prefill chunk
        dict(name="silu_int8_decode_5", path="silu", rows=5, hidden=28672, dtype="bf16", quant="int8"),
        dict(name="silu_fp8_prefill_3001", path="silu", rows=3001, hidden=18432, dtype="bf16", quant="fp8"),
        # int8 projections: one token; a decode batch behind its norm; a prefill chunk's down projection; a full chunk
        dict(name="linear_decode_1", path="linear", m=1, n=8192, k=8192, dtype="bf16", front="rows", bias=False),
        dict(name="linear_norm_decode_23", path="linear", m=23, n=10240, k=8192, dtype="bf16", front="norm", bias=False),
        dict(name="linear_silu_prefill_1000", path="linear", m=1000, n=8192, k=28672, dtype="bf16", front="silu", bias=True),
        dict(name="linear_prefill_4096", path="linear", m=4096, n=10240, k=8192, dtype="f16", front="rows", bias=False),
        # expert layers of one to four decoded tokens, small, medium and large experts
        dict(name="moe_int8_decode_1", path="moe", tokens=1, experts=64, topk=6, hidden=4096, inter=1536, dtype="bf16", quant="int8"),
        dict(name="moe_fp8_decode_3", path="moe", tokens=3, experts=128, topk=8, hidden=2048, inter=768, dtype="bf16", quant="fp8"),
        dict(name="moe_fp8_decode_4", path="moe", tokens=4, experts=256, topk=8, hidden=7168, inter=2048, dtype="f16", quant="fp8"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _times(rng, low, high, step):
    return max(low, min(high, _log(rng, low, high) // step * step))


def draw(rng):
    path = rng.choice(["norm", "norm", "silu", "silu", "linear", "linear", "linear", "moe", "moe"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if path in ("norm", "silu"):
        # row lengths of all kinds: most a multiple of 16 or 8, some odd
        hidden = _times(rng, 16, 16384 if path == "norm" else 28672, rng.choice([16, 16, 16, 8, 1]))
        case = dict(path=path, rows=min(_log(rng, 1, 16384), 4096 * 8192 // hidden), hidden=hidden, dtype=dtype,
                    quant=rng.choice(["fp8", "fp8", "int8", "int8", "static"]))
        if path == "norm":
            case.update(residual=rng.random() < 0.7, y=rng.random() < 0.3, gamma=rng.choice(["same", "same", "f32"]))
        return case
    if path == "linear":
        m, n, k = _log(rng, 1, 4096), _times(rng, 64, 32768, 8), _times(rng, 64, 16384, 16)
        if rng.random() < 0.4:
            n, k = rng.choice([(10240, 8192), (8192, 8192), (8192, 28672), (7168, 16384), (24576, 1536)])
        m = max(1, min(m, 4096 * 10240 * 8192 // (n * k)))
        return dict(path=path, m=m, n=n, k=k, dtype=dtype, front=rng.choice(["rows", "rows", "norm", "silu"]), bias=rng.random() < 0.4)
    experts = rng.choice([8, 16, 32, 64, 128, 256])
    return dict(path=path, tokens=_log(rng, 1, 4), experts=experts, topk=rng.randint(1, 8), hidden=_times(rng, 512, 7168, 128),
                inter=_times(rng, 128, 2048, 128), dtype=dtype, quant=rng.choice(["int8", "fp8"]))


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
class _Maker:
    """Tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32, std=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=dtype).mul_(std)

    def uniform(self, *shape, low, high):
        return torch.rand(*shape, generator=self.g, device="cuda").mul_(high - low).add_(low)

    def weight(self, *shape, int8):
        """8-bit codes of a normally distributed weight whose rows fill the range, slice by slice."""
        out = torch.empty(shape, device="cuda", dtype=torch.int8 if int8 else F8)
        flat, peak = out.view(-1), 127.0 if int8 else 448.0
        for at in range(0, flat.numel(), 1 << 28):
            part = flat[at:at + (1 << 28)]
            part.copy_(self.normal(part.numel(), dtype=torch.bfloat16, std=peak / 4).clamp_(-peak, peak))
        return out

    def scales(self, *shape):
        return self.uniform(*shape, low=1.2e-4, high=2.4e-4)  # weights of standard deviation near 0.02

    def gamma(self, n, dtype):
        return self.uniform(n, low=0.5, high=1.5).to(dtype)


def prepare(case, seed):
    make, dtype, path = _Maker(seed), DTYPES[case["dtype"]], case["path"]
    s = dict(case=case, dtype=dtype)
    if path == "norm":
        rows, hidden = case["rows"], case["hidden"]
        s.update(x=make.normal(rows, hidden, dtype=dtype), gamma=make.gamma(hidden, torch.float32 if case["gamma"] == "f32" else dtype),
                 residual=make.normal(rows, hidden, dtype=dtype, std=2.0) if case["residual"] else None)
    elif path == "silu":
        rows, hidden = case["rows"], case["hidden"]
        s.update(x=make.normal(rows, 2 * hidden, dtype=dtype, std=1.5))
    elif path == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        if case["front"] == "norm":
            s.update(x=make.normal(m, k, dtype=dtype), gamma=make.gamma(k, dtype), residual=make.normal(m, k, dtype=dtype, std=2.0))
        elif case["front"] == "silu":
            s.update(x=make.normal(m, 2 * k, dtype=dtype, std=1.5))
        else:
            # what a one-sided activation leaves: small negative values, large positive ones
            s.update(x=torch.nn.functional.gelu(make.normal(m, k, std=2.0)).to(dtype))
        w = make.weight(n, k, int8=True)
        s.update(w=w, wscale=make.scales(n, 1), wsums=torch.sum(w, dim=1, dtype=torch.int32),
                 bias=make.normal(n, dtype=dtype, std=0.1) if case["bias"] else None)
    else:
        t, e, k, h, i = (case[key] for key in ("tokens", "experts", "topk", "hidden", "inter"))
        int8 = case["quant"] == "int8"
        chosen = torch.topk(torch.softmax(make.normal(t, e), dim=-1), min(k, e), dim=-1)
        codes, hscale = (_plain_int8 if int8 else _plain_fp8)(make.normal(t, h))
        s.update(x=codes.to(torch.int8 if int8 else F8), xscale=hscale, ids=chosen.indices.to(torch.int32),
                 weights=chosen.values / chosen.values.sum(dim=-1, keepdim=True), w13=make.weight(e, 2 * i, h, int8=int8),
                 w2=make.weight(e, h, i, int8=int8), s13=make.scales(e, 2 * i, 1), s2=make.scales(e, h, 1))
    if case.get("quant") == "static":
        s["scale"] = torch.full((1,), 5.0 / 448.0, device="cuda")
    if case.get("quant") == "int8" and path in ("norm", "silu"):
        s["values"] = torch.empty(case["rows"], case["hidden"], device="cuda", dtype=dtype)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain form: elementary operations in 32 bits
# ---------------------------------------------------------------------------------------------------------------------
def _round_away(v):
    return torch.sign(v) * torch.floor(v.abs() + 0.5)


def _plain_rms(s):
    v = s["x"].float()
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v, v * torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + EPS) * s["gamma"].float()


def _plain_silu(s):
    gate, up = s["x"].float().chunk(2, dim=-1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _plain_fp8(y, scale=None):
    scale = y.abs().amax(dim=-1, keepdim=True) / 448.0 if scale is None else scale.expand(y.shape[0], 1)
    mul = torch.where(scale == 0, torch.zeros_like(scale), 1.0 / scale)
    return (y * mul).clamp(-448.0, 448.0).to(F8), scale


def _plain_int8(y):
    amax = y.abs().amax(dim=-1, keepdim=True).clamp_min(1e-10)
    return _round_away(y * (127.0 / amax)), amax / 127.0


def _plain_asym(y):
    lo, hi = y.amin(dim=-1, keepdim=True).clamp_max(0.0), y.amax(dim=-1, keepdim=True).clamp_min(0.0)
    scale = (hi - lo).clamp_min(1e-10) / 255.0
    zp = torch.round(-128.0 - lo / scale)
    return (torch.round(y / scale) + zp).clamp(-128.0, 127.0), scale, zp


def _plain_rows(s, y):
    """The 8-bit outputs of norm and silu: codes (e4m3) or the values that they stand for (int8), and the scales."""
    if s["case"]["quant"] == "int8":
        codes, scale = _plain_int8(y)
        return dict(values=(codes * scale).to(s["dtype"]), scale=scale)
    codes, scale = _plain_fp8(y, s.get("scale"))
    return dict(codes=codes, scale=scale)


def _plain_norm(s):
    v, y = _plain_rms(s)
    out = _plain_rows(s, y)
    if s["case"]["residual"]:
        out["residual"] = v.to(s["dtype"])
    if s["case"]["y"]:
        out["y"] = y.to(s["dtype"])
    return out


def _plain_linear(s):
    front = s["case"]["front"]
    out = {}
    if front == "norm":
        v, y = _plain_rms(s)
        out["residual"] = v.to(s["dtype"])
    else:
        y = _plain_silu(s) if front == "silu" else s["x"].float()
    codes, scale, zp = _plain_asym(y)
    out["out"] = torch.matmul(codes - zp, s["w"].float().t()) * (scale * s["wscale"].view(1, -1))
    if s["bias"] is not None:
        out["out"] = out["out"] + s["bias"].float()
    out["out"] = out["out"].to(s["dtype"])
    return out


def _plain_moe(s):
    case, dtype = s["case"], s["dtype"]
    rows8 = _plain_int8 if case["quant"] == "int8" else _plain_fp8
    pair = s["ids"].long().view(-1)

    def product(codes, w, scale, wscale):
        chosen = w.view(torch.uint8)[pair].view(w.dtype).float()
        return torch.matmul(chosen, codes.float().unsqueeze(-1)).squeeze(-1) * (scale * wscale[pair].squeeze(-1))

    topk = s["ids"].shape[1]
    h = product(s["x"].float().repeat_interleave(topk, dim=0), s["w13"], s["xscale"].repeat_interleave(topk, dim=0), s["s13"])
    gate, up = h.chunk(2, dim=-1)
    codes, scale = rows8(gate / (1.0 + torch.exp(-gate)) * up)
    rows = product(codes, s["w2"], scale, s["s2"]) * s["weights"].view(-1, 1)
    return dict(out=rows.view(-1, topk, rows.shape[-1]).sum(dim=1).to(dtype))


# ---------------------------------------------------------------------------------------------------------------------
# the library's operators
# ---------------------------------------------------------------------------------------------------------------------
def _own_rows(s, q):
    if s["case"]["quant"] == "int8":
        # (int8 codes are compared as the values that they stand for)
        return dict(values=torch.mul(q[0], q[1], out=s["values"]), scale=q[1])
    return dict(codes=q[0], scale=q[1])


def _own_norm(s):
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant

    case = s["case"]
    q, y, residual = fused_rms_row_quant(s["x"], s["gamma"], EPS, res=s["residual"], dtype_quant=torch.int8 if case["quant"] == "int8" else F8,
                                         scale=s.get("scale"), output_unquantized=case["y"])
    out = _own_rows(s, q)
    if case["residual"]:
        out["residual"] = residual
    if case["y"]:
        out["y"] = y
    return out


def _own_silu(s):
    from sglang_amd.quantization.fused_row_quant import silu_and_mul_row_quant

    return _own_rows(s, silu_and_mul_row_quant(s["x"], dtype_quant=torch.int8 if s["case"]["quant"] == "int8" else F8, scale=s.get("scale")))


def _own_linear(s):
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant, silu_and_mul_row_quant
    from sglang_amd.quantization.int8_utils import apply_int8_linear

    front, w = s["case"]["front"], s["w"].t()
    if front == "rows":
        return dict(out=apply_int8_linear(s["x"], w, s["wscale"], weight_sums=s["wsums"], bias=s["bias"]))
    out = {}
    if front == "norm":
        (q, scale, zp), _, out["residual"] = fused_rms_row_quant(s["x"], s["gamma"], EPS, res=s["residual"], dtype_quant=torch.int8, symmetric=False)
    else:
        q, scale, zp = silu_and_mul_row_quant(s["x"], dtype_quant=torch.int8, symmetric=False)
    out["out"] = apply_int8_linear(q, w, s["wscale"], weight_sums=s["wsums"], input_scale=scale, input_zero_point=zp, bias=s["bias"],
                                   out_dtype=s["dtype"])
    return out


def _own_moe(s):
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens

    return dict(out=fused_experts_few_tokens(s["x"], s["xscale"], s["w13"], s["w2"], s["s13"], s["s2"], s["weights"], s["ids"],
                                             out_dtype=s["dtype"]))


def run(state):
    path = state["case"]["path"]
    if own:
        if path == "norm":
            return _own_norm(state)
        if path == "silu":
            return _own_silu(state)
        return _own_linear(state) if path == "linear" else _own_moe(state)
    if path == "norm":
        return _plain_norm(state)
    if path == "silu":
        return _plain_rows(state, _plain_silu(state))
    return _plain_linear(state) if path == "linear" else _plain_moe(state)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _near(v):
    """The nearest whole number, halves away from zero."""
    return torch.where(v < 0, torch.ceil(v - 0.5), torch.floor(v + 0.5))


def _codes_e4m3(v):
    """The e4m3 numbers nearest to v, |v| <= 448: three bits behind the leading one, 2^-6 the smallest normal one's."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))).clamp(-6, 8) - 3)
    return torch.round(v / step) * step


def _exact_8bit(y, kind, scale=None):
    if kind == "int8":
        scale = torch.clamp(y.abs().max(dim=-1, keepdim=True).values, min=1e-10) / 127
        return _near(y / scale), scale
    scale = (y.abs().max(dim=-1, keepdim=True).values / 448) if scale is None else scale.double().repeat(y.shape[0], 1)
    safe = torch.where(scale == 0, torch.ones_like(scale), scale)
    return _codes_e4m3((y / safe).clamp(-448, 448)), scale


def _exact_normed(s):
    v = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
    return v, v / torch.sqrt(torch.sum(v * v, dim=-1, keepdim=True) / v.shape[-1] + EPS) * s["gamma"].double()


def _exact_act(x):
    half = x.shape[-1] // 2
    return x[:, :half] * torch.sigmoid(x[:, :half]) * x[:, half:]


def exact(case, seed):
    s = prepare(case, seed)
    path, dtype = case["path"], DTYPES[case["dtype"]]
    if path in ("norm", "silu"):
        out = {}
        if path == "norm":
            v, y = _exact_normed(s)
            if case["residual"]:
                out["residual"] = v
            if case["y"]:
                out["y"] = y
        else:
            y = _exact_act(s["x"].double())
        codes, out["scale"] = _exact_8bit(y, case["quant"], s.get("scale"))
        if case["quant"] == "int8":
            out["values"] = codes * out["scale"]
        else:
            out["codes"] = codes
        return out
    if path == "linear":
        out = {}
        if case["front"] == "norm":
            out["residual"], y = _exact_normed(s)
        else:
            y = _exact_act(s["x"].double()) if case["front"] == "silu" else s["x"].double()
        low = torch.clamp(y.min(dim=-1, keepdim=True).values, max=0)
        scale = torch.clamp(torch.clamp(y.max(dim=-1, keepdim=True).values, min=0) - low, min=1e-10) / 255
        zp = torch.round(-128 - low / scale)
        centred = torch.clamp(torch.round(y / scale) + zp, -128, 127) - zp
        out["out"] = centred @ s["w"].double().t() * scale * s["wscale"].double().view(1, -1)
        if s["bias"] is not None:
            out["out"] += s["bias"].double()
        return out
    # one (token, expert) pair after the other
    out = torch.zeros(case["tokens"], case["hidden"], device="cuda", dtype=torch.float64)
    half = case["inter"]
    for t in range(case["tokens"]):
        for j, e in enumerate(s["ids"][t].tolist()):
            h = (s["w13"][e].double() @ s["x"][t].double()) * s["xscale"][t].double() * s["s13"][e, :, 0].double()
            codes, scale = _exact_8bit((h[:half] * torch.sigmoid(h[:half]) * h[half:]).view(1, -1), case["quant"])
            out[t] += (s["w2"][e].double() @ codes[0]) * scale[0] * s["s2"][e, :, 0].double() * s["weights"][t, j].double()
    return dict(out=out)


def work(case):
    path = case["path"]
    if path in ("norm", "silu"):
        rows, hidden = case["rows"], case["hidden"]
        read = 4 if path == "silu" or case["residual"] else 2
        moved = rows * (hidden * (read + 1) + 4)
        if path == "norm":
            moved += rows * hidden * (2 * case["residual"] + 2 * case["y"]) + hidden * (4 if case["gamma"] == "f32" else 2)
        return dict(bytes=moved, flops=0)
    if path == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        front = {"rows": 2 * m * k, "norm": 6 * m * k + 2 * k, "silu": 4 * m * k}[case["front"]]
        return dict(bytes=front + n * k + 8 * n + 2 * m * n + (2 * n if case["bias"] else 0), flops=2.0 * m * n * k)
    t, e, h, i = case["tokens"], case["experts"], case["hidden"], case["inter"]
    topk = min(case["topk"], e)
    active = e * (1.0 - (1.0 - topk / e) ** t)  # experts that at least one token is expected to pick
    return dict(bytes=active * (3 * h * i + 4 * (2 * i + h)) + 3 * t * h, flops=6.0 * t * topk * h * i)
