"""Calls that the contracts of rotations, appends and gathers allow, in combinations that a model may make: caches of two types, a norm
without a rotation, one weight of two, operands that are expanded or strided, pools whose rows have one head, inference mode."""
import pytest
import torch

from sglang_amd import append_kv, append_latent, gather_kv, gather_latent, norm_rotate_qk, rotate_qk
from tests.head_rows import check_16, heads, normed, table, turned
from tests.test_kv_cache_gpu import BF16, EPS, F16, KINDS, check_cache, gathered, make_cache, make_slots

pytestmark = pytest.mark.gpu

T, HQ, HK, DIM, PAGES, PAGE = 11, 6, 2, 128, 5, 8


@pytest.mark.parametrize("k_kind", KINDS)
@pytest.mark.parametrize("v_kind", KINDS)
def test_keys_and_values_of_different_types(dev, k_kind, v_kind):
    g = torch.Generator().manual_seed(70)
    k, v = heads(g, T, HK, DIM, dtype=F16).cuda(), heads(g, T, HK, 72, dtype=F16).cuda()
    (kc, ks), (vc, vs) = make_cache(g, k_kind, PAGES, PAGE, (HK, DIM), F16), make_cache(g, v_kind, PAGES, PAGE, (HK, 72), F16, "heads")
    before = [None if t is None else t.clone() for t in (kc, ks, vc, vs)]
    slots, positions, cos_sin = make_slots(g, T, PAGES, PAGE, ((3, -1),)).cuda(), torch.randint(0, 90, (T,), generator=g).int().cuda(), table(90, 64).cuda()
    assert append_kv(k, v, kc, vc, slots, k_scale=ks, v_scale=vs, positions=positions, cos_sin=cos_sin) == (None, None)
    check_cache(kc, before[0], ks, before[1], slots, *turned(*normed(k, None, EPS), positions, cos_sin, False), k_kind, PAGES * PAGE)
    check_cache(vc, before[2], vs, before[3], slots, *normed(v, None, EPS), v_kind, PAGES * PAGE)
    back = gather_kv(kc, vc, slots, F16, k_scale=ks, v_scale=vs)
    for rows, cache, scale, dim in ((back[0], kc, ks, DIM), (back[1], vc, vs, 72)):
        assert torch.equal(rows.cpu(), gathered(cache, scale, slots, F16, PAGES * PAGE, (HK, dim)))


@pytest.mark.parametrize("which", ["q", "k", "both"])
@pytest.mark.parametrize("rotated", [False, True])
@pytest.mark.parametrize("dim", [128, 72, 90])
def test_norms_without_rotations_and_one_of_two(dev, dim, rotated, which):
    g = torch.Generator().manual_seed(71 + dim)
    q, k, v = (heads(g, T, h, dim, dtype=BF16).cuda() for h in (HQ, HK, HK))
    kc, vc = (torch.zeros(PAGES * PAGE, HK, dim, device=dev, dtype=BF16) for _ in range(2))
    wq = (torch.rand(dim, generator=g) + 0.5).to(BF16).cuda() if which != "k" else None
    wk = (torch.rand(dim, generator=g) + 0.5).cuda() if which != "q" else None
    slots = torch.randperm(PAGES * PAGE, generator=g)[:T].cuda()
    turn = dict(positions=torch.randint(0, 90, (T,), generator=g).cuda(), cos_sin=table(90, dim).cuda()) if rotated else {}
    if wq is None and not rotated:
        q = None
    got, none = append_kv(k, v, kc, vc, slots, q=q, q_weight=wq, k_weight=wk, epsilon=EPS, **turn)
    assert none is None and (got is None) == (q is None)

    def want(x, w):
        y = normed(x, w, EPS)
        return turned(*y, turn["positions"], turn["cos_sin"], False) if rotated else y

    if q is not None:
        check_16(got, *want(q, wq))
    check_16(kc[slots], *want(k, wk))
    assert torch.equal(vc[slots], v)


@pytest.mark.parametrize("dim", [128, 72, 90])
def test_expanded_and_strided_operands(dev, dim):
    """One key head that stands for several, one position for all axes, every other slot, scales and weights between other numbers."""
    g = torch.Generator().manual_seed(72 + dim)
    one = heads(g, T, 1, dim, dtype=BF16).cuda()
    k = one.expand(T, 3, dim)
    v = heads(g, 1, 3, dim, dtype=BF16).cuda().expand(T, 3, dim)
    slots = torch.randperm(PAGES * PAGE, generator=g)[:2 * T].cuda()[::2]
    positions = torch.randint(0, 90, (2 * T,), generator=g).cuda()[1::2].expand(3, T)
    half = dim // 2
    turn = dict(sections=[half - 2 * (half // 3), half // 3, half // 3], alternating=True)
    turn["cos_sin"] = torch.cat([table(90, dim).cuda(), torch.ones(90, 6, device=dev)], dim=1)[:, :dim]
    scales = (torch.rand(9, generator=g) * 0.02 + 0.005).cuda()
    k_scale, v_scale = scales[::3], scales[1:2]
    caches = [make_cache(g, "e4m3", PAGES, PAGE, (3, dim), BF16, "heads")[0] for _ in range(2)]
    before = [c.clone() for c in caches]
    assert k_scale.stride(0) == 3
    append_kv(k, v, caches[0], caches[1], slots, k_scale=k_scale, v_scale=v_scale, positions=positions, **turn)
    wanted = turned(*normed(k, None, EPS), positions, turn["cos_sin"], False, turn["sections"], True)
    check_cache(caches[0], before[0], k_scale, None, slots, *wanted, "e4m3", PAGES * PAGE)
    check_cache(caches[1], before[1], v_scale, None, slots, *normed(v, None, EPS), "e4m3", PAGES * PAGE)
    back = gather_kv(caches[0], caches[1], slots, BF16, k_scale=k_scale, v_scale=v_scale)
    assert torch.equal(back[0].cpu(), gathered(caches[0], k_scale, slots, BF16, PAGES * PAGE, (3, dim)))
    assert torch.equal(back[1].cpu(), gathered(caches[1], v_scale, slots, BF16, PAGES * PAGE, (3, dim)))


def test_pools_of_rows_with_one_head(dev):
    """A pool [slots, 1, 512 + 64], as a page of one slot each, and the same rows without that dimension."""
    g = torch.Generator().manual_seed(73)
    latent, rope, q = heads(g, T, 512, dtype=BF16).cuda(), heads(g, T, 64, dtype=BF16).cuda(), heads(g, T, HQ, 64, dtype=BF16).cuda()
    slots, positions, cos_sin = torch.randperm(40, generator=g)[:T].cuda(), torch.randint(0, 90, (T,), generator=g).cuda(), table(90, 64).cuda()
    weight = (torch.rand(512, generator=g) + 0.5).to(BF16).cuda()
    pool, flat = torch.zeros(40, 1, 576, device=dev, dtype=BF16), torch.zeros(40, 576, device=dev, dtype=BF16)
    got = [append_latent(latent, rope, p[..., :512], p[..., 512:], slots, positions, cos_sin, weight=weight, epsilon=EPS, q_rope=q) for p in (pool, flat)]
    assert torch.equal(got[0], got[1]) and torch.equal(pool.squeeze(1), flat)
    check_16(flat[slots, :512], *normed(latent, weight, EPS))
    assert torch.equal(gather_latent(pool[..., :512], pool[..., 512:], slots, BF16), flat[slots])


def test_no_heads(dev):
    """Tensors without heads beside ones that have some."""
    g = torch.Generator().manual_seed(74)
    positions, cos_sin, slots = torch.arange(T, device=dev), table(20, 64).cuda(), torch.arange(T, device=dev)
    x, none = heads(g, T, HK, 64, dtype=BF16).cuda(), torch.empty(T, 0, 64, device=dev, dtype=BF16)
    for q, k in ((x, none), (none, x), (none, none)):
        got = rotate_qk(q, k, positions, cos_sin)
        for a, b in zip(got, (q, k)):
            assert a.shape == b.shape
            if b.numel():
                check_16(a, *turned(*normed(b, None, EPS), positions, cos_sin, False))
    cache, empty = torch.zeros(20, HK, 64, device=dev, dtype=BF16), torch.zeros(20, 0, 64, device=dev, dtype=BF16)
    append_kv(none, x, empty, cache, slots)
    assert torch.equal(cache[:T], x) and not cache[T:].any()
    k, v = gather_kv(empty, cache, slots, BF16)
    assert k.shape == none.shape and torch.equal(v, x)
    v, k = gather_kv(cache, empty, slots, BF16)
    assert k.shape == none.shape and torch.equal(v, x)


def test_inference_mode_and_parameters(dev):
    g = torch.Generator().manual_seed(75)
    q, k = heads(g, T, HQ, 64, dtype=BF16).cuda(), heads(g, T, HK, 64, dtype=BF16).cuda()
    w = torch.nn.Parameter((torch.rand(64, generator=g) + 0.5).cuda())
    positions, cos_sin = torch.arange(T, device=dev), table(20, 64).cuda()
    with pytest.raises(NotImplementedError):
        norm_rotate_qk(q, k, w, w, EPS, positions, cos_sin)
    with torch.no_grad():
        want = norm_rotate_qk(q, k, w, w, EPS, positions, cos_sin)
    with torch.inference_mode():
        cache = torch.zeros(20, HK, 64, device=dev, dtype=BF16)
        got = norm_rotate_qk(q, k, w, w, EPS, positions, cos_sin)
        append_kv(k, k, cache, torch.zeros_like(cache), positions, k_weight=w, epsilon=EPS, positions=positions, cos_sin=cos_sin)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        cast = norm_rotate_qk(q, k, w, w, EPS, positions, cos_sin)
    for a in (got, cast):
        assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1])
    assert torch.equal(cache[:T], want[1])


def test_a_prompt_captured_with_new_outputs(dev):
    """Replays of a captured prompt chunk whose queries go into a tensor of the graph's own, on a stream of its own."""
    g = torch.Generator().manual_seed(76)
    qkv = torch.zeros(300, HQ + 2 * HK, DIM, device=dev, dtype=BF16)
    positions, slots, cos_sin = torch.zeros(300, device=dev, dtype=torch.int32), torch.zeros(300, device=dev, dtype=torch.int32), table(500, DIM).cuda()
    (kc, ks), (vc, vs) = (make_cache(g, "e4m3_rows", 50, 8, (HK, DIM), BF16) for _ in range(2))
    eager = [t.clone() for t in (kc, ks, vc, vs)]
    slots.copy_(torch.randperm(400, generator=g)[:300])

    def put(a, b, c, d):
        return append_kv(qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:], a, c, slots, k_scale=b, v_scale=d, q=qkv[:, :HQ], positions=positions, cos_sin=cos_sin)[0]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        put(kc, ks, vc, vs)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = put(kc, ks, vc, vs)
    put(*eager)
    for _ in range(4):
        qkv.copy_(heads(g, 300, HQ + 2 * HK, DIM, dtype=BF16))
        positions.copy_(torch.randint(0, 500, (300,), generator=g))
        slots.copy_(torch.randperm(400, generator=g)[:300])
        graph.replay()
        want = put(*eager)
        torch.cuda.synchronize()
        assert torch.equal(q, want)
        for a, b in zip((kc, ks, vc, vs), eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
