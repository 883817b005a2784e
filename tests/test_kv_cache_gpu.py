"""Appends to paged caches and gathers from them against their definitions in 64 bits."""
import pytest
import torch

from sglang_amd import append_kv, append_latent, gather_kv, gather_latent, norm_rotate_qk, rotate_qk
from tests.head_rows import F8, check_16, check_8, heads, normed, table, turned

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
EPS = 1e-6
KINDS = ["16", "e4m3", "e4m3_heads", "e4m3_rows", "int8_rows"]


def bits(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def make_cache(g, kind, pages, page, rows, dtype, layout="tokens", flat=False):
    """(cache [pages, page, *rows] with earlier contents, its type's row scales or None)."""
    h = rows[0] if len(rows) == 2 else None
    shape = (pages, page, *rows) if layout == "tokens" else (pages, h, page, rows[1])
    if kind == "16":
        cache = torch.randn(*shape, generator=g).to(dtype)
    elif kind.startswith("int8"):
        cache = torch.randint(-127, 128, shape, generator=g).to(torch.int8)
    else:
        cache = (torch.randn(*shape, generator=g) * 50).to(F8)
    cache = cache.cuda()
    scale = None
    if kind == "e4m3":
        scale = torch.full((1,), 0.0213).cuda()
    elif kind == "e4m3_heads":
        scale = (torch.rand(h, generator=g) * 0.02 + 0.005).cuda()
    elif kind.endswith("_rows"):
        scale = (torch.rand(shape[:-1], generator=g) + 0.5).cuda()
    if layout == "heads":
        cache = cache.transpose(1, 2)
        scale = scale.transpose(1, 2) if kind.endswith("_rows") else scale
    if flat:
        cache = cache.reshape(pages * page, *rows)
        scale = scale.reshape(pages * page, h) if kind.endswith("_rows") else scale
    return cache, scale


def make_slots(g, tokens, pages, page, padding=()):
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    for at, value in padding:
        if at < tokens:
            slots[at] = value
    return slots


def check_cache(cache, before, scale, scale_before, slots, want, off, kind, total, group=None):
    """The rows of the slots against their 64-bit values, all other rows and scales as they were."""
    slots = slots.cpu().long()
    kept = (slots >= 0) & (slots < total)
    at = slots[kept]
    flat = lambda t, rows: t.cpu().reshape(total, *rows)  # noqa: E731
    rows = want.shape[1:]
    now, old = flat(bits(cache), rows), flat(bits(before), rows)
    rest = torch.ones(total, dtype=torch.bool)
    rest[at] = False
    assert torch.equal(now[rest], old[rest]), "rows of other slots changed"
    got = now[at].view(cache.dtype) if cache.element_size() == 1 else now[at]
    want, off = want[kept], off[kept]
    if kind == "16":
        check_16(got, want, off)
    elif scale.dim() <= 1:
        check_8(got, want, off, given=scale.cpu().double().view(-1, 1))
    else:
        lead = rows[:-1] if group is None else (scale.shape[-1],)
        new, was = flat(scale, lead), flat(scale_before, lead)
        assert torch.equal(new[rest], was[rest]), "scales of other slots changed"
        s = new[at].unsqueeze(-1) if group is None else new[at]
        check_8(got, want, off, scales=s, group=group)


def run_append(tokens, hq, hk, dim, dim_v, width, kind, page, layout="tokens", norm=False, dtype=BF16, interleaved=False, flat=False, index=torch.int64,
               padding=((1, -1), (4, 10 ** 9)), seed=0):
    g = torch.Generator().manual_seed(tokens * 100 + dim + seed)
    q, k, v = (heads(g, tokens, h, d, dtype=dtype).cuda() for h, d in ((hq, dim), (hk, dim), (hk, dim_v)))
    pages = tokens // page + 3
    caches = [make_cache(g, kind, pages, page, (hk, d), dtype, layout, flat) for d in (dim, dim_v)]
    before = [(c.clone(), None if s is None else s.clone()) for c, s in caches]
    slots = make_slots(g, tokens, pages, page, padding).to(index).cuda()
    positions, cos_sin = torch.randint(0, 300, (tokens,), generator=g).to(index).cuda(), table(300, width).cuda()
    wq, wk = ((torch.rand(dim, generator=g) + 0.5).cuda() for _ in range(2)) if norm else (None, None)
    k_out = torch.empty_like(k)
    got, back = append_kv(k, v, caches[0][0], caches[1][0], slots, k_scale=caches[0][1], v_scale=caches[1][1], q=q, positions=positions,
                          cos_sin=cos_sin, interleaved=interleaved, q_weight=wq, k_weight=wk, epsilon=EPS, k_out=k_out)
    assert back.data_ptr() == k_out.data_ptr()
    total = pages * page
    wanted = [turned(*normed(x, w, EPS), positions, cos_sin, interleaved) for x, w in ((q, wq), (k, wk))] + [normed(v, None, EPS)]
    check_16(got, *wanted[0])
    check_16(k_out, *wanted[1])
    for i in range(2):
        check_cache(caches[i][0], before[i][0], caches[i][1], before[i][1], slots, *wanted[1 + i], kind, total)
    return caches, slots


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [(1, 8, 1, 128, 128, 128), (6, 8, 2, 64, 64, 32), (7, 6, 3, 80, 80, 80), (5, 3, 3, 72, 72, 72), (9, 4, 1, 90, 90, 90),
                                  (3, 4, 2, 192, 128, 64), (70, 5, 5, 256, 256, 256), (2, 2, 1, 2, 2, 2), (5, 1, 1, 1024, 512, 64), (3, 1, 1, 1022, 38, 38)])
def test_append(dev, size, kind):
    for page, layout, norm in ((16, "tokens", True), (5, "heads", False), (1, "tokens", False)):
        run_append(*size, kind, page, layout, norm)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_forms(dev, dtype, kind):
    run_append(12, 4, 2, 128, 128, 128, kind, 1, dtype=dtype, flat=True, index=torch.int32, interleaved=True)
    run_append(12, 4, 2, 128, 128, 64, kind, 64, dtype=dtype, interleaved=True, norm=True, layout="heads")
    run_append(12, 4, 2, 72, 128, 72, kind, 7, dtype=dtype, interleaved=True, norm=True)


@pytest.mark.parametrize("kind", KINDS)
def test_append_many(dev, kind):
    run_append(1030, 61, 7, 128, 128, 128, kind, 16, norm=kind == "16")
    run_append(1030, 61, 7, 72, 72, 72, kind, 16, norm=kind != "16")


@pytest.mark.parametrize("kind", ["16", "int8_rows"])
def test_gather_many(dev, kind):
    """Launches of four units a lane: 17000 rows of 2 x 8 x 128."""
    g = torch.Generator().manual_seed(21)
    caches = [make_cache(g, kind, 100, 16, (8, 128), BF16) for _ in range(2)]
    slots = torch.randint(-1, 1601, (17000,), generator=g).cuda()
    got = gather_kv(caches[0][0], caches[1][0], slots, BF16, k_scale=caches[0][1], v_scale=caches[1][1])
    for rows, (cache, scale) in zip(got, caches):
        assert torch.equal(rows.cpu(), gathered(cache, scale, slots, BF16, 1600, (8, 128)))


def test_keys_and_values_alone(dev):
    """No rotation, no queries: values and keys are copied bit for bit, from one projection's rows into the halves of one buffer."""
    g = torch.Generator().manual_seed(2)
    kv = heads(g, 6, 4, 64, dtype=BF16).cuda()
    kv[0, 0, 0], kv[1, 3, 5], kv[2, 1, 2] = float("inf"), float("nan"), -0.0
    both = torch.zeros(5, 2, 4, 2, 64, device=dev, dtype=BF16)
    slots = torch.tensor([3, 19, 0, 7, 12, -5], device=dev)
    assert append_kv(kv[:, :2], kv[:, 2:], both[:, 0], both[:, 1], slots) == (None, None)
    want = torch.zeros_like(both)
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            want[s // 4, 0, s % 4], want[s // 4, 1, s % 4] = kv[t, :2], kv[t, 2:]
    assert torch.equal(both.isnan(), want.isnan()) and torch.equal(both.nan_to_num(1.5).view(torch.int16), want.nan_to_num(1.5).view(torch.int16))


@pytest.mark.parametrize("kind", ["e4m3_rows", "int8_rows", "e4m3"])
def test_bad_values_stay_in_their_row(dev, kind):
    g = torch.Generator().manual_seed(3)
    v = heads(g, 4, 2, 64, dtype=BF16).cuda()
    v[1, 0, 7], v[2, 1, 3], v[3, 0] = float("nan"), float("inf"), 0
    caches = [make_cache(g, kind, 2, 4, (2, 64), BF16) for _ in range(2)]
    slots = torch.arange(4, device=dev)
    append_kv(v, v, caches[0][0], caches[1][0], slots, k_scale=caches[0][1], v_scale=caches[1][1])
    cache, scale = caches[1]
    back = gather_kv(caches[0][0], cache, slots, BF16, k_scale=caches[0][1], v_scale=scale)[1]
    if kind == "e4m3":
        assert torch.isnan(back).nonzero().tolist() == [[1, 0, 7]] and (back[2, 1, 3] > 0).all()
    else:
        assert torch.isnan(scale[0, 1, 0]) and torch.isinf(scale[0, 2, 1]) and torch.isfinite(scale[0, 0]).all()
        assert torch.isnan(back[1, 0]).all() and not torch.isfinite(back[2, 1]).any()
    assert torch.isfinite(back[0]).all() and (back[3, 0] == 0).all() and torch.isfinite(back[3, 1]).all()
    if kind == "int8_rows":
        assert (scale[0, 3, 0] - 1e-10 / 127).abs() < 1e-18
    if kind == "e4m3_rows":
        assert scale[0, 3, 0] == 0


LATENT = [(1, 1, 512, 64), (5, 16, 512, 64), (7, 3, 256, 32), (3, 2, 128, 10), (4, 2, 384, 64), (2, 2, 1024, 64), (3, 1, 640, 6), (6, 2, 72, 8)]


@pytest.mark.parametrize("kind", ["16", "e4m3", "e4m3_groups", "e4m3_row", "int8_groups"])
@pytest.mark.parametrize("size", LATENT)
def test_latent(dev, size, kind):
    tokens, hq, c, r = size
    if kind.endswith("_groups") and c % 128:
        kind = kind.replace("_groups", "_row")
    for page, norm, interleaved, dtype in ((16, True, True, BF16), (1, False, False, F16), (5, True, False, BF16)):
        g = torch.Generator().manual_seed(tokens * 10 + c)
        row = heads(g, tokens, c + r, dtype=dtype).cuda()
        latent, rope = row[:, :c], row[:, c:]
        q = heads(g, tokens, hq, 16 + r, dtype=dtype).cuda()[:, :, 16:]
        pages = tokens // page + 3
        if kind in ("16", "e4m3"):
            whole, scale = make_cache(g, kind, pages, page, (c + r,), dtype)
            cache, rope_cache, rope_scale = whole[..., :c], whole[..., c:], scale
        else:
            cache, _ = make_cache(g, kind, pages, page, (c,), dtype)
            scale = torch.rand(pages, page, 1 if kind.endswith("_row") else c // 128, generator=g).cuda()
            rope_cache, rope_scale = make_cache(g, "16", pages, page, (r,), dtype)
        before, rope_before, scale_before = cache.clone(), rope_cache.clone(), None if scale is None else scale.clone()
        slots = make_slots(g, tokens, pages, page, ((2, -1),)).cuda()
        positions, cos_sin = torch.randint(0, 300, (tokens,), generator=g).cuda(), table(300, r).cuda()
        w = (torch.rand(c, generator=g) + 0.5).to(dtype).cuda() if norm else None
        got = append_latent(latent, rope, cache, rope_cache, slots, positions, cos_sin, weight=w, epsilon=EPS, interleaved=interleaved, scale=scale,
                            rope_scale=rope_scale, q_rope=q)
        check_16(got, *turned(*normed(q, None, EPS), positions, cos_sin, interleaved))
        group = None
        if kind not in ("16", "e4m3"):
            group = c if kind.endswith("_row") else 128
        check_cache(cache, before, scale, scale_before, slots, *normed(latent, w, EPS), kind, pages * page, group)
        want, off = turned(*normed(rope.unsqueeze(1), None, EPS), positions, cos_sin, interleaved)
        check_cache(rope_cache, rope_before, rope_scale, None, slots, want.squeeze(1), off.squeeze(1), "16" if rope_scale is None else "e4m3", pages * page)


def gathered(cache, scale, slots, dtype, total, rows, group=None):
    """code * scale in 32 bits, rounded once: bit for bit."""
    slots = slots.cpu().long()
    inside = (slots >= 0) & (slots < total)
    at = slots.clamp(0, total - 1)
    values = cache.cpu().reshape(total, *rows) if cache.element_size() == 2 else bits(cache).cpu().reshape(total, *rows).view(cache.dtype)
    got = values[at] if cache.element_size() == 2 else values.view(torch.uint8)[at].view(cache.dtype).float()
    if scale is not None:
        s = scale.cpu().view(-1, 1) if scale.dim() <= 1 else scale.cpu().reshape(total, -1)[at]
        if group is not None:
            s = s.repeat_interleave(group, dim=-1)
        elif scale.dim() > 1:
            s = s.unsqueeze(-1)
        got = got * s
    got = got.to(dtype)
    got[~inside] = 0
    return got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,h,dim", [(1, 1, 128), (37, 8, 128), (5, 3, 72), (4, 2, 90), (3, 2, 36), (9, 1, 1024), (2, 5, 7), (6, 2, 1), (3000, 8, 128)])
def test_gather(dev, rows, h, dim, kind):
    g = torch.Generator().manual_seed(rows + dim)
    for page, layout, dtype, index in ((16, "tokens", BF16, torch.int64), (7, "heads", F16, torch.int32)):
        pages = max(rows // page // 2, 1)
        caches = [make_cache(g, kind, pages, page, (h, dim), dtype, layout) for _ in range(2)]
        slots = torch.randint(0, pages * page, (2 * rows,), generator=g)[::2].to(index)  # the same slot more than once
        if rows > 2:
            slots[1], slots[2] = -1, pages * page
        slots = slots.cuda()
        wide = torch.full((rows, h, dim + 5), 3.0, device=dev, dtype=dtype)
        v_out = wide[..., 2:2 + dim]
        k, v = gather_kv(caches[0][0], caches[1][0], slots, dtype, k_scale=caches[0][1], v_scale=caches[1][1], v_out=v_out)
        assert v.data_ptr() == v_out.data_ptr() and (wide[..., :2] == 3).all() and (wide[..., 2 + dim:] == 3).all()
        for got, (cache, scale) in zip((k, v), caches):
            assert torch.equal(got.cpu(), gathered(cache, scale, slots, dtype, pages * page, (h, dim)))


@pytest.mark.parametrize("kind", ["16", "e4m3", "e4m3_groups", "e4m3_row", "int8_groups"])
@pytest.mark.parametrize("rows,c,r", [(1, 512, 64), (515, 512, 64), (7, 128, 10), (3, 256, 6)])
def test_gather_latent(dev, rows, c, r, kind):
    g = torch.Generator().manual_seed(rows + c)
    pages, page = rows // 16 + 1, 16
    cache, scale = make_cache(g, kind, pages, page, (c,), BF16)
    rope_cache, rope_scale = make_cache(g, kind if kind in ("16", "e4m3") else "16", pages, page, (r,), BF16)
    group = None
    if kind not in ("16", "e4m3"):
        group = c if kind.endswith("_row") else 128
        scale = torch.rand(pages, page, c // group, generator=g).cuda()
    slots = torch.randint(-1, pages * page + 1, (rows,), generator=g).cuda()
    got = gather_latent(cache, rope_cache, slots, BF16, scale=scale, rope_scale=rope_scale)
    total = pages * page
    assert torch.equal(got[:, :c].cpu(), gathered(cache, scale, slots, BF16, total, (c,), group))
    assert torch.equal(got[:, c:].cpu(), gathered(rope_cache, rope_scale, slots, BF16, total, (r,)))
    wide = torch.full((rows, c + r + 3), 3.0, device=dev, dtype=BF16)
    out = gather_latent(cache, rope_cache, slots, BF16, scale=scale, rope_scale=rope_scale, out=wide[:, 1:1 + c + r])
    assert torch.equal(out, got) and (wide[:, 0] == 3).all() and (wide[:, 1 + c + r:] == 3).all()


def test_offsets_beyond_32_bits(dev):
    """Slots whose rows lie more than 2^32 bytes into a cache, and into its scales."""
    slots_count, h, dim = (1 << 32) // (2 * 1024) + 100, 2, 1024  # e4m3 rows of 2 KB: a little over 4 GiB
    cache = torch.zeros(slots_count, h, dim, device=dev, dtype=torch.int8)
    small = torch.zeros(slots_count, 1, 2, device=dev, dtype=torch.int8)
    scale, small_scale = torch.zeros(slots_count, h, device=dev), torch.zeros(slots_count, 1, device=dev)
    g = torch.Generator().manual_seed(4)
    k, v = heads(g, 3, h, dim, dtype=BF16).cuda(), heads(g, 3, 1, 2, dtype=BF16).cuda()
    slots = torch.tensor([slots_count - 1, 5, slots_count - 50], device=dev)
    append_kv(k, v, cache, small, slots, k_scale=scale, v_scale=small_scale)
    assert int((cache.view(-1, h * dim).ne(0).any(dim=1)).sum()) == 3
    check_8(cache[slots].cpu(), *normed(k, None, EPS), scales=scale[slots].unsqueeze(-1))
    back, _ = gather_kv(cache, small, slots, BF16, k_scale=scale, v_scale=small_scale)
    assert torch.equal(back, (cache[slots].float() * scale[slots].unsqueeze(-1)).to(BF16))


def test_no_tokens(dev):
    cos_sin = table(10, 64).cuda()
    none, slots = torch.empty(0, 2, 64, device=dev, dtype=BF16), torch.empty(0, device=dev, dtype=torch.int64)
    cache = torch.ones(3, 2, 64, device=dev, dtype=BF16)
    q, _ = append_kv(none, none, cache, cache.clone(), slots, q=none, positions=slots, cos_sin=cos_sin)
    assert q.shape == none.shape and (cache == 1).all()
    k, v = gather_kv(cache, cache, slots, BF16)
    assert k.shape == v.shape == none.shape
    no_cache = torch.empty(0, 2, 64, device=dev, dtype=BF16)  # a cache without slots takes nothing
    append_kv(torch.ones(2, 2, 64, device=dev, dtype=BF16), torch.ones(2, 2, 64, device=dev, dtype=BF16), no_cache, no_cache.clone(),
              torch.tensor([0, 1], device=dev))
    assert (gather_kv(no_cache, no_cache, torch.tensor([0, 1], device=dev), BF16)[0] == 0).all()


def test_a_prompt_and_its_decoded_tokens(dev):
    """As a layer would use them: a prompt in two chunks and decoded tokens into one int8 cache of shuffled pages, by captured
    replays, the context read back and compared with the rows that went in."""
    g = torch.Generator().manual_seed(11)
    hq, hk, dim, page, pages, dtype = 8, 2, 128, 16, 12, BF16
    order = torch.randperm(pages, generator=g)
    place = lambda p: order[p // page] * page + p % page  # noqa: E731
    cos_sin = table(256, dim).cuda()
    wq, wk = (torch.rand(dim, generator=g) + 0.5).cuda(), (torch.rand(dim, generator=g) + 0.5).cuda()
    caches = [make_cache(g, "int8_rows", pages, page, (hk, dim), dtype, "heads") for _ in range(2)]
    (kc, ks), (vc, vs) = caches
    kept_k, kept_v = [], []

    def put(qkv, positions, slots, q_out=None):
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        return append_kv(k, v, kc, vc, slots, k_scale=ks, v_scale=vs, q=q, positions=positions, cos_sin=cos_sin, q_weight=wq, k_weight=wk, epsilon=EPS,
                         q_out=q_out)[0]

    for start, n in ((0, 37), (37, 60)):
        qkv, positions = heads(g, n, hq + 2 * hk, dim, dtype=dtype).cuda(), torch.arange(start, start + n)
        q = put(qkv, positions.cuda(), place(positions).cuda())
        want = norm_rotate_qk(qkv[:, :hq], qkv[:, hq:hq + hk], wq, wk, EPS, positions.cuda(), cos_sin)
        assert torch.equal(q, want[0])
        kept_k.append(want[1]), kept_v.append(qkv[:, hq + hk:])
    # single tokens, with two rows of padding in the captured batch
    qkv = torch.zeros(3, hq + 2 * hk, dim, device=dev, dtype=dtype)
    positions, slots = torch.zeros(3, dtype=torch.int64, device=dev), torch.full((3,), -1, device=dev)
    q_out = torch.empty(3, hq, dim, device=dev, dtype=dtype)
    put(qkv, positions, slots, q_out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        put(qkv, positions, slots, q_out)
    for p in range(97, 103):
        qkv.copy_(heads(g, 3, hq + 2 * hk, dim, dtype=dtype))
        positions[0], slots[0] = p, place(torch.tensor(p)).item()
        graph.replay()
        torch.cuda.synchronize()
        want = norm_rotate_qk(qkv[:1, :hq], qkv[:1, hq:hq + hk], wq, wk, EPS, positions[:1], cos_sin)
        assert torch.equal(q_out[:1], want[0])
        kept_k.append(want[1]), kept_v.append(qkv[:1, hq + hk:].clone())
    context = place(torch.arange(103)).cuda()
    k, v = gather_kv(kc, vc, context, dtype, k_scale=ks, v_scale=vs)
    for got, rows in ((k, torch.cat(kept_k)), (v, torch.cat(kept_v))):
        rows = rows.cpu().double()
        step = rows.abs().amax(dim=-1, keepdim=True) / 127
        # half a step of int8; the rows that went in, their scale and the rows that came back are each rounded to bfloat16 or finer
        assert ((got.cpu().double() - rows).abs() <= step * (0.5 + 2.0 ** -7) + rows.abs() * 2.0 ** -7 * (1 + 2.0 ** -7)).all()
    # both together are what the parts are
    alone = rotate_qk(qkv[:, :hq], qkv[:, hq:hq + hk], positions, cos_sin)
    fresh = torch.zeros(8, hk, dim, device=dev, dtype=dtype)
    q, _ = append_kv(qkv[:, hq:hq + hk], qkv[:, hq + hk:], fresh, torch.zeros_like(fresh), torch.arange(3, device=dev), q=qkv[:, :hq], positions=positions,
                     cos_sin=cos_sin)
    assert torch.equal(q, alone[0]) and torch.equal(fresh[:3], alone[1]) and not fresh[3:].any()


def test_latent_rows_of_one_buffer(dev):
    """A slot as bytes: 512 codes, four scales, the rotary part in 16 bits; appended and read back."""
    g = torch.Generator().manual_seed(12)
    raw = torch.zeros(10, 16, 512 + 16 + 128, dtype=torch.uint8, device=dev)
    cache = raw[..., :512].view(F8)
    scale, rope_cache = raw[..., 512:528].view(torch.float32), raw[..., 528:].view(BF16)
    latent, rope = heads(g, 20, 512, dtype=BF16).cuda(), heads(g, 20, 64, dtype=BF16).cuda()
    slots, positions, cos_sin = torch.randperm(160, generator=g)[:20].cuda(), torch.arange(20, device=dev), table(32, 64).cuda()
    append_latent(latent, rope, cache, rope_cache, slots, positions, cos_sin, scale=scale)
    back = gather_latent(cache, rope_cache, slots, BF16, scale=scale)
    groups = latent.cpu().double().view(20, 4, 128)
    off = (back[:, :512].cpu().double().view(20, 4, 128) - groups).abs()
    # half a step of e4m3 among normal numbers, of its smallest ones below, and of bfloat16
    bound = groups.abs() * (2.0 ** -4 + 2.0 ** -7) + groups.abs().amax(dim=-1, keepdim=True) / 448 * 2.0 ** -10 * 1.01
    assert (off <= bound).all()
    assert torch.equal(back[:, 512:].unsqueeze(1), rotate_qk(rope.unsqueeze(1), None, positions, cos_sin)[0])
    rest = torch.ones(160, dtype=torch.bool, device=dev)
    rest[slots] = False
    assert not raw.view(160, -1)[rest].any()


def test_in_place(dev):
    """Queries and keys rotated in their own buffer, a view of the projection, while they go into the cache."""
    g = torch.Generator().manual_seed(14)
    qkv = heads(g, 9, 8, 64, dtype=BF16).cuda()
    before = qkv.clone()
    positions, cos_sin, slots = torch.randint(0, 50, (9,), generator=g).cuda(), table(50, 64).cuda(), torch.randperm(20, generator=g)[:9].cuda()
    caches = [torch.zeros(20, 2, 64, device=dev, dtype=BF16) for _ in range(2)]
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    got = append_kv(k, v, *caches, slots, q=q, positions=positions, cos_sin=cos_sin, q_out=q, k_out=k)
    assert got[0].data_ptr() == q.data_ptr() and got[1].data_ptr() == k.data_ptr()
    check_16(q, *turned(*normed(before[:, :4], None, EPS), positions, cos_sin, False))
    check_16(k, *turned(*normed(before[:, 4:6], None, EPS), positions, cos_sin, False))
    assert torch.equal(v, before[:, 6:]) and torch.equal(caches[0][slots], k) and torch.equal(caches[1][slots], v)


def test_two_streams_into_one_cache(dev):
    g = torch.Generator().manual_seed(15)
    k = heads(g, 2, 400, 8, 128, dtype=BF16).cuda()
    slots = torch.randperm(1000, generator=g)[:800].view(2, 400).cuda()
    (kc, ks), (vc, vs) = (make_cache(g, "int8_rows", 125, 8, (8, 128), BF16) for _ in range(2))
    want = [t.clone() for t in (kc, ks, vc, vs)]
    for i in range(2):
        append_kv(k[i], k[i], want[0], want[2], slots[i], k_scale=want[1], v_scale=want[3])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            append_kv(k[i], k[i], kc, vc, slots[i], k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    for got, ref in zip((kc, ks, vc, vs), want):
        assert torch.equal(got, ref)


def test_the_same_slot_twice(dev):
    """Either of the two rows, or parts of both; all other rows as they were."""
    k = torch.stack([torch.full((2, 64), 1.0), torch.full((2, 64), 2.0), torch.full((2, 64), 3.0)]).to(BF16).cuda()
    cache = torch.zeros(6, 2, 64, device=dev, dtype=BF16)
    append_kv(k, k, cache, torch.zeros_like(cache), torch.tensor([4, 1, 4], device=dev))
    assert ((cache[4] == 1) | (cache[4] == 3)).all() and (cache[1] == 2).all() and not cache[[0, 2, 3, 5]].any()


def test_gradients_are_refused(dev):
    leaf = torch.ones(3, 2, 64, device=dev, dtype=BF16, requires_grad=True)
    x, cache, slots = torch.ones(3, 2, 64, device=dev, dtype=BF16), torch.zeros(6, 2, 64, device=dev, dtype=BF16), torch.arange(3, device=dev)
    with pytest.raises(NotImplementedError, match="no gradient"):
        append_kv(leaf, x, cache, cache.clone(), slots)
    with pytest.raises(NotImplementedError, match="no gradient"):
        append_kv(x, x, cache, torch.zeros(6, 2, 64, device=dev, dtype=BF16, requires_grad=True), slots)
    with pytest.raises(NotImplementedError, match="no gradient"):
        gather_kv(cache, torch.zeros(6, 2, 64, device=dev, dtype=BF16, requires_grad=True), slots, BF16)
    assert not cache.any()
    version = cache._version
    append_kv(x, x, cache, cache.clone(), slots)
    assert cache._version == version + 1


def test_behind_a_quantised_projection(dev):
    """A layer's input as this library runs it: residual, norm and int8 codes, the int8 qkv product, heads into an int8 cache, the
    context back.  The heads' values are the product's own output, rounded to int8 rows once."""
    from sglang_amd.quantization.fused_row_quant import fused_rms_row_quant
    from sglang_amd.quantization.int8_utils import apply_int8_linear, int8_weight_sums

    g = torch.Generator().manual_seed(16)
    tokens, hidden, hq, hk, dim = 21, 1024, 8, 2, 128
    x, res = (torch.randn(tokens, hidden, generator=g).to(BF16).cuda() for _ in range(2))
    gamma = (torch.rand(hidden, generator=g) + 0.5).to(BF16).cuda()
    w = torch.randint(-127, 128, ((hq + 2 * hk) * dim, hidden), generator=g).to(torch.int8).cuda()
    wscale = (torch.rand(w.shape[0], 1, generator=g) * 1e-4 + 1e-4).cuda()
    (q8, s8, zp), _, _ = fused_rms_row_quant(x, gamma, EPS, res=res, symmetric=False)
    qkv = apply_int8_linear(q8, w.t(), wscale, weight_sums=int8_weight_sums(w.t()), input_scale=s8, input_zero_point=zp, out_dtype=BF16)
    qkv = qkv.view(tokens, hq + 2 * hk, dim)
    (kc, ks), (vc, vs) = (make_cache(g, "int8_rows", 4, 16, (hk, dim), BF16) for _ in range(2))
    slots, positions, cos_sin = torch.randperm(64, generator=g)[:tokens].cuda(), torch.arange(tokens, device=dev), table(64, dim).cuda()
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    q_out, _ = append_kv(k, v, kc, vc, slots, k_scale=ks, v_scale=vs, q=q, positions=positions, cos_sin=cos_sin)
    check_16(q_out, *turned(*normed(q, None, EPS), positions, cos_sin, False))
    want = turned(*normed(k, None, EPS), positions, cos_sin, False)[0], v.cpu().double()
    for got, rows in zip(gather_kv(kc, vc, slots, BF16, k_scale=ks, v_scale=vs), want):
        step = rows.abs().amax(dim=-1, keepdim=True) / 127
        # half a step of int8, half a step of bfloat16; 2^-20 for the scale and the rotation
        assert ((got.cpu().double() - rows).abs() <= (step * 0.5 * (1 + 2.0 ** -8) + rows.abs() * 2.0 ** -8) * (1 + 2.0 ** -20) + step * 2.0 ** -13).all()
