"""What lies between a layer's first projection and its attention, as cases that can be prepared, run in a plain form or through
this library, and priced.

  rotate  rotary positions applied to the heads of queries and keys; a token's position is one number, or one per axis (time,
          height, width) of an image or a video, each axis turning its own share of the pairs.
  norm    RMSNorm of every query and key head, and the rotation of the normalised heads.
  append  keys (rotated, normalised where asked) and values of new tokens into the slots of a paged cache, and the rotated
          queries: caches in 16 bits, in e4m3 with a scale known beforehand, in e4m3 or int8 with a scale per token and head.
  latent  the same for a cache of compressed rows: RMSNorm of the latent row, rotation of the part that carries the position,
          both into the cache, the queries' rotary parts; latents in 16 bits, e4m3, or e4m3 with a scale per 128 values.
  gather  rows of a paged cache back in 16 bits, in the order of a context: what attention over earlier tokens is fed with.

Definitions (x real, i.e. nothing is rounded unless it says so; round() is to nearest):

  norm     y = x / sqrt(mean(x^2) + eps) * gamma, over one head
  rotate   pair i of a head, (a, b) = (x[i], x[i + R / 2]) ("halves") or (x[2 i], x[2 i + 1]) ("pairs"), i < R / 2, with c and s the
           cosine and sine of pair i in the table's row for the token's position (on the axis of pair i):
           (a, b) becomes (a c - b s, b c + a s);  the values behind the first R stay
  axes     "blocks": the first sections[0] pairs belong to axis 0, the next sections[1] to axis 1, and so on;  "alternating": pair
           i to axis a = i mod A where i < A sections[a], to axis 0 otherwise
  e4m3     code = e4m3(clamp(y / scale, -448, 448)), scale as given or max|y| / 448 of the head (of 128 values of a latent)
  int8     amax = max(max|y|, 1e-10);  scale = amax / 127;  code = round(y / scale)
  slot     a token's row is row slot % page of page slot / page; tokens of a negative slot (padding) write nothing
  gather   out = code * scale

Sizes are those of the benchmark's DeepSeek-V3 and Llama-3-70B layers and generic ones."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
F8 = torch.float8_e4m3fn
EPS = 1e-6


def listed():
    llama = dict(heads=64, kv_heads=8, dim=128, rotary=128, style="halves")
    return [
        # one decoded token: queries and keys of a Llama-3-70B layer
        dict(name="rotate_decode_1", path="rotate", tokens=1, **llama, axes="one", dtype="bf16"),
        # a prompt with an image in it: three axes, ragged length
        dict(name="rotate_image_2901", path="rotate", tokens=2901, heads=28, kv_heads=4, dim=128, rotary=128, style="halves", axes="blocks", dtype="bf16"),
        # the rotary parts of a DeepSeek-V3 prefill chunk's queries, views into rows of 192 values a head
        dict(name="rotate_parts_4096", path="rotate", tokens=4096, heads=128, kv_heads=1, dim=64, rotary=64, style="pairs", axes="one", dtype="bf16"),
        # a ragged decode batch whose heads are normalised; then a prefill chunk with a video, half of each head rotated
        dict(name="norm_decode_37", path="norm", tokens=37, heads=32, kv_heads=4, dim=128, rotary=128, style="halves", axes="one", gamma="f32", dtype="f16"),
        dict(name="norm_video_4096", path="norm", tokens=4096, heads=64, kv_heads=8, dim=128, rotary=64, style="halves", axes="alternating", gamma="same", dtype="bf16"),
        # one decoded token into an e4m3 cache; a padded decode batch into int8 rows, and the context read back; a prefill chunk
        dict(name="append_decode_1", path="append", tokens=1, **llama, axes="one", norm=False, cache="e4m3", page=16, layout="tokens", mode="decode", dtype="bf16"),
        dict(name="append_int8_decode_61", path="append", tokens=61, **llama, axes="one", norm=True, cache="int8_rows", page=64, layout="heads", mode="decode", dtype="bf16"),
        dict(name="append_prefill_8191", path="append", tokens=8191, **llama, axes="one", norm=False, cache="e4m3_rows", page=16, layout="tokens", mode="prefill", dtype="bf16"),
        # the latent cache of a DeepSeek-V3 layer: a decode batch in 16 bits, a prefill chunk in e4m3 with a scale per 128 values
        dict(name="latent_decode_128", path="latent", tokens=128, heads=128, latent=512, rotary=64, style="pairs", cache="16", page=64, mode="decode", dtype="bf16"),
        dict(name="latent_prefill_4095", path="latent", tokens=4095, heads=128, latent=512, rotary=64, style="pairs", cache="e4m3_groups", page=64, mode="prefill", dtype="bf16"),
        # contexts for attention in 16 bits: a short one of latents, a long one of int8 rows
        dict(name="gather_latent_515", path="gather", rows=515, kind="latent", heads=1, dim=512, rotary=64, cache="e4m3_groups", page=64, dtype="bf16"),
        dict(name="gather_int8_65000", path="gather", rows=65000, kind="kv", heads=8, dim=128, rotary=0, cache="int8_rows", page=16, dtype="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    kv = rng.choice([1, 1, 2, 4, 5, 8, 8])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256, 72])
    return dict(heads=min(kv * rng.choice([1, 2, 4, 6, 7, 8]), 64), kv_heads=kv, dim=dim, rotary=dim if dim == 72 else rng.choice([dim, dim, dim // 2]))


def draw(rng):
    path = rng.choice(["rotate", "rotate", "norm", "norm", "append", "append", "append", "latent", "latent", "gather", "gather"])
    case = dict(path=path, dtype=rng.choice(["bf16", "bf16", "f16"]))
    if path == "latent":
        mode = rng.choice(["decode", "prefill"])
        case.update(tokens=_log(rng, 1, 512 if mode == "decode" else 4095), heads=rng.choice([8, 16, 32, 64, 128]), latent=rng.choice([256, 512, 512, 512]),
                    rotary=rng.choice([32, 64, 64]), style=rng.choice(["pairs", "pairs", "halves"]),
                    cache=rng.choice(["16", "e4m3", "e4m3_groups"]), page=rng.choice([1, 16, 64]), mode=mode)
        return case
    if path == "gather":
        kind = rng.choice(["kv", "kv", "latent"])
        if kind == "latent":
            case.update(rows=_log(rng, 1, 65000), kind=kind, heads=1, dim=512, rotary=64, cache=rng.choice(["16", "e4m3", "e4m3_groups"]))
        else:
            case.update(rows=_log(rng, 1, 65000), kind=kind, heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 80, 96, 128, 128]), rotary=0,
                        cache=rng.choice(["16", "e4m3", "e4m3_rows", "int8_rows"]))
        case.update(page=rng.choice([1, 16, 64]))
        return case
    case.update(tokens=_log(rng, 1, 8191), **_heads(rng), style=rng.choice(["halves", "halves", "pairs"]))
    case["tokens"] = max(1, min(case["tokens"], 4096 * 9216 // ((case["heads"] + 2 * case["kv_heads"]) * case["dim"])))
    case["axes"] = rng.choice(["one", "one", "blocks", "alternating"])
    if path == "norm":
        case.update(gamma=rng.choice(["same", "same", "f32"]))
    if path == "append":
        mode = rng.choice(["decode", "prefill"])
        case.update(axes="one", norm=rng.random() < 0.4, cache=rng.choice(["16", "e4m3", "e4m3_rows", "int8_rows"]), page=rng.choice([1, 16, 16, 64]),
                    layout=rng.choice(["tokens", "tokens", "heads"]), mode=mode)
        if mode == "decode":
            case["tokens"] = min(case["tokens"], 512)
    return case


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _sections(case):
    """How many pairs turn with each of three axes: a quarter with time and the rest shared, or nearly even ones."""
    half = case["rotary"] // 2
    if case["axes"] == "blocks":
        t = max(half // 4, 1)
        return [t, (half - t) // 2, half - t - (half - t) // 2]
    third = half // 3
    return [half - 2 * third, third, third]


def _pair_axes(case):
    half, sections = case["rotary"] // 2, _sections(case)
    if case["axes"] == "blocks":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [i % 3 if i < 3 * sections[i % 3] else 0 for i in range(half)]


class _Maker:
    """Tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32, std=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=dtype).mul_(std)

    def uniform(self, *shape, low, high):
        return torch.rand(*shape, generator=self.g, device="cuda").mul_(high - low).add_(low)

    def below(self, high, *shape):
        return torch.randint(0, high, shape, generator=self.g, device="cuda")

    def permutation(self, n):
        return torch.argsort(torch.rand(n, generator=self.g, device="cuda"))

    def heads(self, *shape, dtype):
        """Heads as a projection leaves them: some channels much larger than others."""
        return self.normal(*shape).mul_(torch.exp(self.normal(shape[-1], std=0.7))).to(dtype)

    def gamma(self, n, dtype):
        return self.uniform(n, low=0.5, high=1.5).to(dtype)

    def table(self, rows, rotary, base=500000.0):
        """cosines | sines of every position, the angles in 64 bits."""
        turn = torch.arange(rows, device="cuda", dtype=torch.float64).view(-1, 1) * torch.pow(
            base, torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / -rotary)
        return torch.cat([torch.cos(turn), torch.sin(turn)], dim=-1).float()

    def image_positions(self, tokens):
        """Text, a grid of pictures' patches in three axes, text again."""
        text = tokens // 8
        side = max(int(math.sqrt(max(tokens - 2 * text, 1) / 2)), 1)
        i = torch.arange(tokens, device="cuda")
        patch = (i - text).clamp_min(0)
        grid = torch.stack([patch // (side * side), patch // side % side, patch % side]) + text
        inside = (i >= text) & (i < tokens - text)
        behind = i - (tokens - text) + text + side
        return torch.where(inside, grid, torch.where(i < text, i, behind).expand(3, -1)).contiguous()

    def codes(self, *shape, int8):
        if int8:
            return self.below(255, *shape).sub_(127).to(torch.int8)
        return self.normal(*shape, dtype=torch.bfloat16, std=100.0).clamp_(-448, 448).to(F8)

    def cache(self, kind, *shape, dtype):
        """A cache that holds earlier tokens."""
        if kind == "16":
            return self.normal(*shape, dtype=dtype)
        return self.codes(*shape, int8=kind.startswith("int8"))

    def scales(self, *shape):
        return self.uniform(*shape, low=0.01, high=0.05)


def _slots(make, case, s):
    """Slots of the new tokens in a cache of shuffled pages, and of a whole context in its order."""
    tokens, page = case["tokens"], case["page"]
    if case["mode"] == "decode":
        # each sequence has pages of its own and writes somewhere in its last one
        pages = tokens + max(1024 // page, 1)
        order = make.permutation(pages)
        slots = order[:tokens] * page + make.below(page, tokens)
        positions = make.below(8192, tokens)
        if tokens > 8:  # a batch padded to a size that has been captured
            slots[-3:] = -1
            positions[-3:] = 0
    else:
        # the second chunk of a prompt: it begins inside a page
        start = 1000 + page // 2
        pages = (start + tokens) // page + 2
        order = make.permutation(pages)
        positions = torch.arange(tokens, device="cuda") + start
        slots = order[positions // page] * page + positions % page
    s.update(slots=slots, positions=positions, pages=pages)
    s["context"] = (order.view(-1, 1) * page + torch.arange(page, device="cuda")).view(-1)


def prepare(case, seed):
    make, dtype, path = _Maker(seed), DTYPES[case["dtype"]], case["path"]
    s = dict(case=case, dtype=dtype)
    if path == "gather":
        rows, page, h, d, r, kind = (case[key] for key in ("rows", "page", "heads", "dim", "rotary", "cache"))
        pages = rows // page + 17
        order = make.permutation(pages)
        at = torch.arange(rows, device="cuda")
        s["slots"] = order[at // page] * page + at % page
        if case["kind"] == "latent":
            s["latent_cache"] = make.cache(kind, pages, page, d, dtype=dtype)
            s["rope_cache"] = make.cache("16" if kind == "e4m3_groups" else kind, pages, page, r, dtype=dtype)
            s["scale"] = {"16": None, "e4m3": make.scales(1), "e4m3_groups": make.scales(pages, page, d // 128)}[kind]
            s["rope_scale"] = s["scale"] if kind == "e4m3" else None
            s["out"] = torch.empty(rows, d + r, device="cuda", dtype=dtype)
            return s
        for name in ("k", "v"):
            s[name + "_cache"] = make.cache(kind, pages, page, h, d, dtype=dtype)
            s[name + "_scale"] = None if kind == "16" else make.scales(1) if kind == "e4m3" else make.scales(pages, page, h)
            s[name + "_out"] = torch.empty(rows, h, d, device="cuda", dtype=dtype)
        return s
    t = case["tokens"]
    if path == "latent":
        h, c, r, page = case["heads"], case["latent"], case["rotary"], case["page"]
        _slots(make, case, s)
        row = make.heads(t, c + r, dtype=dtype)  # one row of a down projection
        q = make.heads(t, h, 128 + r, dtype=dtype)
        s.update(latent=row[:, :c], rope=row[:, c:], q_rope=q[:, :, 128:], q_out=torch.empty(t, h, r, device="cuda", dtype=dtype), gamma=make.gamma(c, dtype))
        kind = case["cache"]
        if kind == "e4m3_groups":
            s.update(latent_cache=make.cache(kind, s["pages"], page, c, dtype=dtype), rope_cache=make.cache("16", s["pages"], page, r, dtype=dtype),
                     scale=make.scales(s["pages"], page, c // 128), rope_scale=None)
        else:
            rows = make.cache(kind, s["pages"], page, c + r, dtype=dtype)  # latent and rotary part of a slot lie side by side
            s.update(latent_cache=rows[..., :c], rope_cache=rows[..., c:], scale=None if kind == "16" else torch.full((1,), 0.02, device="cuda"))
            s["rope_scale"] = s["scale"]
        s["cos_sin"] = make.table(8192 + 1024, r, base=10000.0)
        return s
    h, kv, d, r = (case[key] for key in ("heads", "kv_heads", "dim", "rotary"))
    if d == 64 and h == 128:
        # rotary parts: the last 64 of 192 values of a query head, the last 64 of a row of latents
        s.update(q=make.heads(t, h, 192, dtype=dtype)[:, :, 128:], k=make.heads(t, 1, 576, dtype=dtype)[:, :, 512:])
    else:
        qkv = make.heads(t, h + 2 * kv, d, dtype=dtype)  # one row of the projection
        s.update(q=qkv[:, :h], k=qkv[:, h:h + kv], v=qkv[:, h + kv:])
    s["q_out"] = torch.empty(t, h, d, device="cuda", dtype=dtype)
    if path == "append":
        _slots(make, case, s)
        page, kind = case["page"], case["cache"]
        for name in ("k", "v"):
            shape = (s["pages"], page, kv) if case["layout"] == "tokens" else (s["pages"], kv, page)
            flip = (lambda x: x) if case["layout"] == "tokens" else (lambda x: x.transpose(1, 2))
            s[name + "_cache"] = flip(make.cache(kind, *shape, d, dtype=dtype))
            s[name + "_scale"] = None if kind == "16" else torch.full((1,), 0.02, device="cuda") if kind == "e4m3" else flip(make.scales(*shape))
            if kind == "int8_rows":
                s[name + "_context"] = torch.empty(s["context"].numel(), kv, d, device="cuda", dtype=dtype)
        s["cos_sin"] = make.table(8192 + 1024, r)
    else:
        s["k_out"] = torch.empty(t, kv, d, device="cuda", dtype=dtype)
        if case["axes"] == "one":
            s["positions"] = make.below(8192, t)
        else:
            s["positions"] = make.image_positions(t)
            s["pair_axis"] = torch.tensor(_pair_axes(case), device="cuda")
        s["cos_sin"] = make.table(8192, r)
    if path == "norm" or case.get("norm"):
        gamma_type = torch.float32 if case.get("gamma") == "f32" else dtype
        s.update(q_gamma=make.gamma(d, gamma_type), k_gamma=make.gamma(d, gamma_type))
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain form: elementary operations in 32 bits
# ---------------------------------------------------------------------------------------------------------------------
def _plain_turn(s):
    """(cosines, sines) of every token's pairs, [tokens, 1, R / 2]."""
    half = s["cos_sin"].shape[1] // 2
    if "pair_axis" in s:
        at, pair = s["positions"][s["pair_axis"]].t(), torch.arange(half, device="cuda")
        return s["cos_sin"][at, pair].unsqueeze(1), s["cos_sin"][at, pair + half].unsqueeze(1)
    rows = s["cos_sin"][s["positions"]].unsqueeze(1)
    return rows[..., :half], rows[..., half:]


def _plain_rotate(x, turn, style):
    cos, sin = turn
    r = 2 * cos.shape[-1]
    y = x.clone()
    first, second = (y[..., :r // 2], y[..., r // 2:r]) if style == "halves" else (y[..., 0:r:2], y[..., 1:r:2])
    a, b = first * cos - second * sin, second * cos + first * sin
    first.copy_(a)
    second.copy_(b)
    return y


def _plain_norm(x, gamma):
    return x if gamma is None else x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * gamma.float()


def _plain_codes(y, kind, scale=None):
    """Codes and scales of the rows of y in the cache's type; a scale that is given counts."""
    if kind.startswith("int8"):
        amax = y.abs().amax(dim=-1, keepdim=True).clamp_min(1e-10)
        v = y * (127.0 / amax)
        return (torch.sign(v) * torch.floor(v.abs() + 0.5)).to(torch.int8), amax / 127.0
    scale = y.abs().amax(dim=-1, keepdim=True) / 448.0 if scale is None else scale
    mul = torch.where(scale == 0, torch.zeros_like(scale), 1.0 / scale)
    return (y * mul).clamp(-448.0, 448.0).to(F8), scale


def _plain_put(cache, s, rows):
    """rows [tokens, ...] into their slots of a paged tensor, the pages [pages, page, ...]."""
    page = cache.shape[1]
    kept = torch.nonzero(s["slots"] >= 0).view(-1)
    slots = s["slots"][kept]
    if cache.dtype == F8:
        cache, rows = cache.view(torch.uint8), rows.view(torch.uint8)
    cache[slots // page, slots % page] = rows[kept]


def _plain_get(cache, scale, slots, dtype):
    page = cache.shape[1]
    at = (slots // page, slots % page)
    rows = cache.view(torch.uint8)[at].view(F8) if cache.dtype == F8 else cache[at]
    if scale is None:
        return rows.to(dtype)
    if scale.dim() == 1:
        return (rows.float() * scale).to(dtype)
    scale = scale[at]
    groups = rows.float().view(*scale.shape, -1)
    return (groups * scale.unsqueeze(-1)).view(rows.shape).to(dtype)


def _plain_append(s):
    case, dtype = s["case"], s["dtype"]
    turn, kind = _plain_turn(s), case["cache"]
    q = _plain_rotate(_plain_norm(s["q"].float(), s.get("q_gamma")), turn, case["style"])
    k = _plain_rotate(_plain_norm(s["k"].float(), s.get("k_gamma")), turn, case["style"])
    out = dict(q=q.to(dtype))
    for name, rows in (("k", k), ("v", s["v"].float())):
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        if kind == "16":
            _plain_put(cache, s, rows.to(dtype))
        elif kind == "e4m3":
            _plain_put(cache, s, _plain_codes(rows, kind, scale)[0])
        else:
            codes, scales = _plain_codes(rows, kind)
            _plain_put(cache, s, codes)
            _plain_put(scale, s, scales.squeeze(-1))
            out[name + "_scale"] = scale
        out[name] = _plain_get(cache, scale, s["context"], dtype) if kind == "int8_rows" else cache
    return out


def _plain_latent(s):
    case, dtype = s["case"], s["dtype"]
    turn, kind = _plain_turn(s), case["cache"]
    out = dict(q=_plain_rotate(s["q_rope"].float(), turn, case["style"]).to(dtype), latent=s["latent_cache"], rope=s["rope_cache"])
    latent = _plain_norm(s["latent"].float(), s["gamma"])
    rope = _plain_rotate(s["rope"].float().unsqueeze(1), turn, case["style"]).squeeze(1)
    if kind == "e4m3_groups":
        codes, scales = _plain_codes(latent.view(latent.shape[0], -1, 128), kind)
        _plain_put(s["latent_cache"], s, codes.view(latent.shape))
        _plain_put(s["scale"], s, scales.squeeze(-1))
        _plain_put(s["rope_cache"], s, rope.to(dtype))
        out["scale"] = s["scale"]
    elif kind == "e4m3":
        _plain_put(s["latent_cache"], s, _plain_codes(latent, kind, s["scale"])[0])
        _plain_put(s["rope_cache"], s, _plain_codes(rope, kind, s["rope_scale"])[0])
    else:
        _plain_put(s["latent_cache"], s, latent.to(dtype))
        _plain_put(s["rope_cache"], s, rope.to(dtype))
    return out


def _plain_gather(s):
    if s["case"]["kind"] == "latent":
        return dict(out=torch.cat([_plain_get(s["latent_cache"], s["scale"], s["slots"], s["dtype"]),
                                   _plain_get(s["rope_cache"], s["rope_scale"], s["slots"], s["dtype"])], dim=-1))
    return {name: _plain_get(s[name + "_cache"], s[name + "_scale"], s["slots"], s["dtype"]) for name in ("k", "v")}


def _plain_heads(s):
    turn, style = _plain_turn(s), s["case"]["style"]
    return {name: _plain_rotate(_plain_norm(s[name].float(), s.get(name + "_gamma")), turn, style).to(s["dtype"]) for name in ("q", "k")}


# ---------------------------------------------------------------------------------------------------------------------
# the library's operators
# ---------------------------------------------------------------------------------------------------------------------
def _own_turn(case):
    if case["axes"] == "one":
        return dict(interleaved=case["style"] == "pairs")
    return dict(interleaved=case["style"] == "pairs", sections=_sections(case), alternating=case["axes"] == "alternating")


def _own_heads(s):
    from sglang_amd.rotary import norm_rotate_qk, rotate_qk

    turn = dict(_own_turn(s["case"]), q_out=s["q_out"], k_out=s["k_out"])
    if s["case"]["path"] == "norm":
        q, k = norm_rotate_qk(s["q"], s["k"], s["q_gamma"], s["k_gamma"], EPS, s["positions"], s["cos_sin"], **turn)
    else:
        q, k = rotate_qk(s["q"], s["k"], s["positions"], s["cos_sin"], **turn)
    return dict(q=q, k=k)


def _own_append(s):
    from sglang_amd.kv_cache import append_kv, gather_kv

    case = s["case"]
    q, _ = append_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"], q=s["q"], positions=s["positions"],
                     cos_sin=s["cos_sin"], interleaved=case["style"] == "pairs", q_weight=s.get("q_gamma"), k_weight=s.get("k_gamma"), epsilon=EPS, q_out=s["q_out"])
    out = dict(q=q, k=s["k_cache"], v=s["v_cache"])
    if case["cache"].endswith("_rows"):
        out.update(k_scale=s["k_scale"], v_scale=s["v_scale"])
    if case["cache"] == "int8_rows":
        out["k"], out["v"] = gather_kv(s["k_cache"], s["v_cache"], s["context"], s["dtype"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                       k_out=s["k_context"], v_out=s["v_context"])
    return out


def _own_latent(s):
    from sglang_amd.kv_cache import append_latent

    q = append_latent(s["latent"], s["rope"], s["latent_cache"], s["rope_cache"], s["slots"], s["positions"], s["cos_sin"], weight=s["gamma"], epsilon=EPS,
                      interleaved=s["case"]["style"] == "pairs", scale=s["scale"], rope_scale=s["rope_scale"], q_rope=s["q_rope"], q_out=s["q_out"])
    out = dict(q=q, latent=s["latent_cache"], rope=s["rope_cache"])
    if s["case"]["cache"] == "e4m3_groups":
        out["scale"] = s["scale"]
    return out


def _own_gather(s):
    from sglang_amd.kv_cache import gather_kv, gather_latent

    if s["case"]["kind"] == "latent":
        return dict(out=gather_latent(s["latent_cache"], s["rope_cache"], s["slots"], s["dtype"], scale=s["scale"], rope_scale=s["rope_scale"], out=s["out"]))
    k, v = gather_kv(s["k_cache"], s["v_cache"], s["slots"], s["dtype"], k_scale=s["k_scale"], v_scale=s["v_scale"], k_out=s["k_out"], v_out=s["v_out"])
    return dict(k=k, v=v)


def run(state):
    path = state["case"]["path"]
    if own:
        return {"append": _own_append, "latent": _own_latent, "gather": _own_gather}.get(path, _own_heads)(state)
    return {"append": _plain_append, "latent": _plain_latent, "gather": _plain_gather}.get(path, _plain_heads)(state)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_rotated(x, s):
    """x [tokens, heads, dim], pair after pair as a complex number."""
    half = s["cos_sin"].shape[1] // 2
    axis = s["pair_axis"] if "pair_axis" in s else torch.zeros(half, dtype=torch.long, device="cuda")
    at = (s["positions"] if s["positions"].dim() == 2 else s["positions"].unsqueeze(0)).index_select(0, axis)  # [pairs, tokens]
    flat = s["cos_sin"].double().reshape(-1)
    index = at * (2 * half) + torch.arange(half, device="cuda").unsqueeze(1)
    unit = torch.complex(flat[index], flat[index + half]).t().unsqueeze(1)
    if s["case"]["style"] == "halves":
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * unit
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], dim=-1)
    z = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) * unit
    return torch.cat([torch.view_as_real(z).flatten(-2), x[..., 2 * half:]], dim=-1)


def _exact_normed(x, gamma):
    if gamma is None:
        return x
    return x / torch.sqrt(torch.sum(x * x, dim=-1, keepdim=True) / x.shape[-1] + EPS) * gamma.double()


def _codes_e4m3(v):
    """The e4m3 numbers nearest to v, |v| <= 448: three bits behind the leading one, 2^-6 the smallest normal one's."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))).clamp(-6, 8) - 3)
    return torch.round(v / step) * step


def _exact_e4m3(y, scale):
    safe = torch.where(scale == 0, torch.ones_like(scale), scale)
    return _codes_e4m3((y / safe).clamp(-448, 448))


def _exact_cache(cache, s, rows):
    """The cache with the new tokens' rows, in 64 bits."""
    out = cache.float().double() if cache.dtype == F8 else cache.double()
    pages, page = cache.shape[:2]
    whole = out.reshape(pages * page, *cache.shape[2:])
    valid = s["slots"] >= 0
    whole = whole.index_copy(0, s["slots"][valid], rows[valid])
    return whole.reshape(cache.shape)


def exact(case, seed):
    s = prepare(case, seed)
    path, kind = case["path"], case.get("cache")
    if path in ("rotate", "norm"):
        return {name: _exact_rotated(_exact_normed(s[name].double(), s.get(name + "_gamma")), s) for name in ("q", "k")}
    if path == "gather":
        def back(cache, scale, width):
            rows = (cache.float().double() if cache.dtype == F8 else cache.double()).flatten(0, 1).index_select(0, s["slots"])
            if scale is None:
                return rows
            by = scale.double().expand(rows.shape[0], 1) if scale.dim() == 1 else scale.double().flatten(0, 1).index_select(0, s["slots"])
            return (rows.reshape(rows.shape[0], by.shape[1], -1) * by.unsqueeze(-1)).reshape(rows.shape)

        if case["kind"] == "latent":
            return dict(out=torch.cat([back(s["latent_cache"], s["scale"], 128), back(s["rope_cache"], s["rope_scale"], None)], dim=1))
        return {name: back(s[name + "_cache"], s[name + "_scale"], case["dim"]) for name in ("k", "v")}
    if path == "latent":
        latent = _exact_normed(s["latent"].double(), s["gamma"])
        rope = _exact_rotated(s["rope"].double().unsqueeze(1), s).squeeze(1)
        out = dict(q=_exact_rotated(s["q_rope"].double(), s))
        if kind == "e4m3_groups":
            groups = latent.reshape(latent.shape[0], -1, 128)
            scale = groups.abs().max(dim=-1).values / 448
            out["scale"] = _exact_cache(s["scale"], s, scale)
            latent = _exact_e4m3(groups, scale.unsqueeze(-1)).reshape(latent.shape)
        elif kind == "e4m3":
            latent, rope = _exact_e4m3(latent, s["scale"].double()), _exact_e4m3(rope, s["scale"].double())
        out["latent"], out["rope"] = _exact_cache(s["latent_cache"], s, latent), _exact_cache(s["rope_cache"], s, rope)
        return out
    out = dict(q=_exact_rotated(_exact_normed(s["q"].double(), s.get("q_gamma")), s))
    new = dict(k=_exact_rotated(_exact_normed(s["k"].double(), s.get("k_gamma")), s), v=s["v"].double())
    for name, rows in new.items():
        cache = s[name + "_cache"]
        if kind == "16":
            out[name] = _exact_cache(cache, s, rows)
        elif kind == "e4m3":
            out[name] = _exact_cache(cache, s, _exact_e4m3(rows, s[name + "_scale"].double()))
        else:
            peak = rows.abs().max(dim=-1, keepdim=True).values
            scale = torch.clamp(peak, min=1e-10) / 127 if kind == "int8_rows" else peak / 448
            out[name + "_scale"] = _exact_cache(s[name + "_scale"], s, scale.squeeze(-1))
            if kind == "int8_rows":
                v = rows / scale
                codes = _exact_cache(cache, s, torch.where(v < 0, torch.ceil(v - 0.5), torch.floor(v + 0.5)))
                out[name] = (codes * out[name + "_scale"].unsqueeze(-1)).flatten(0, 1).index_select(0, s["context"])
            else:
                out[name] = _exact_cache(cache, s, _exact_e4m3(rows, scale))
    return out


def work(case):
    path, kind = case["path"], case.get("cache")
    held = 2 if kind == "16" else 1  # bytes of a cached value
    if path == "gather":
        rows, width = case["rows"], case["heads"] * case["dim"]
        if case["kind"] == "latent":
            rope = case["rotary"] * (2 if kind in ("16", "e4m3_groups") else 1)
            scales = 4 * (case["dim"] // 128) if kind == "e4m3_groups" else 0
            return dict(bytes=rows * (8 + width * held + rope + scales + 2 * (width + case["rotary"])), flops=0)
        scales = 4 * case["heads"] if kind.endswith("_rows") else 0
        return dict(bytes=rows * (8 + 2 * (width * held + scales + 2 * width)), flops=0)
    t, r = case["tokens"], case["rotary"]
    turn = t * (4 * r + 8)  # a row of the table and a position for each token
    if path == "latent":
        rope = 2 if kind == "e4m3_groups" else held
        scales = 4 * (case["latent"] // 128) if kind == "e4m3_groups" else 0
        return dict(bytes=turn + t * (8 + 4 * case["heads"] * r + (2 + held) * case["latent"] + (2 + rope) * r + scales) + 2 * case["latent"], flops=0)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if path == "append":
        moved = turn + t * (8 + 4 * h * d + 2 * kv * d * (2 + held) + (8 * kv if kind.endswith("_rows") else 0))
        if kind == "int8_rows":  # the context read back: its codes, scales and slots, and the 16-bit rows
            page = case["page"]
            pages = t + max(1024 // page, 1) if case["mode"] == "decode" else (1000 + page // 2 + t) // page + 2
            moved += pages * page * (8 + 2 * kv * (3 * d + 4))
        return dict(bytes=moved, flops=0)
    axes = 8 * t * (2 if case["axes"] != "one" else 0)
    return dict(bytes=turn + axes + 4 * t * (h + kv) * d, flops=0)
