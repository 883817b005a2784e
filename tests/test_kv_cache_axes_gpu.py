"""Keys appended to paged caches with positions on several axes, as a model of images or video does, against the definitions in 64 bits and
against the rotation alone."""
import random

import pytest
import torch

from sglang_amd import append_kv, norm_rotate_qk, rotate_qk
from tests.head_rows import check_16, heads, normed, table, turned
from tests.test_heads_random_gpu import sizes
from tests.test_kv_cache_gpu import BF16, EPS, F16, KINDS, check_cache, make_cache, make_slots

pytestmark = pytest.mark.gpu

F32 = torch.float32


def sections_of(half, axes, style):
    """Pairs of up to `axes` axes, uneven ones."""
    axes = min(axes, half)
    share = half // axes
    sections = [half - (axes - 1) * share] + [share] * (axes - 1)
    return sections if style == "alternating" else sections[::-1]


def run(tokens, hq, hk, dim, dim_v, width, kind, style, axes=3, page=16, layout="tokens", norm=False, dtype=BF16, table_dtype=F32, interleaved=False,
        index=torch.int64, padding=((1, -1), (4, 10 ** 9)), seed=0):
    g = torch.Generator().manual_seed(tokens * 100 + dim + seed)
    qkv = heads(g, tokens, hq + hk, dim, dtype=dtype).cuda()
    q, k, v = qkv[:, :hq], qkv[:, hq:], heads(g, tokens, hk, dim_v, dtype=dtype).cuda()
    pages = tokens // page + 3
    caches = [make_cache(g, kind, pages, page, (hk, d), dtype, layout) for d in (dim, dim_v)]
    before = [(c.clone(), None if s is None else s.clone()) for c, s in caches]
    slots = make_slots(g, tokens, pages, page, padding).to(index).cuda()
    sections = sections_of(width // 2, axes, style)
    positions = torch.randint(0, 300, (len(sections), tokens), generator=g)
    positions[:, ::3] = positions[:1, ::3]  # text: the same on every axis
    positions, cos_sin = positions.to(index).cuda(), table(300, width, table_dtype).cuda()
    wq, wk = ((torch.rand(dim, generator=g) + 0.5).cuda() for _ in range(2)) if norm else (None, None)
    turn = dict(interleaved=interleaved, sections=sections, alternating=style == "alternating")
    got, k_out = append_kv(k, v, caches[0][0], caches[1][0], slots, k_scale=caches[0][1], v_scale=caches[1][1], q=q, positions=positions, cos_sin=cos_sin,
                           q_weight=wq, k_weight=wk, epsilon=EPS, k_out=torch.empty_like(k), **turn)
    wanted = [turned(*normed(x, w, EPS), positions, cos_sin, **turn) for x, w in ((q, wq), (k, wk))] + [normed(v, None, EPS)]
    check_16(got, *wanted[0])
    check_16(k_out, *wanted[1])
    for i in range(2):
        check_cache(caches[i][0], before[i][0], caches[i][1], before[i][1], slots, *wanted[1 + i], kind, pages * page)
    alone = norm_rotate_qk(q, k, wq, wk, EPS, positions, cos_sin, **turn) if norm else rotate_qk(q, k, positions, cos_sin, **turn)
    # (bit for bit, but for a norm beside values of another size: they may ask for smaller pieces, whose squares are summed in another order)
    assert (norm and dim_v != dim) or (torch.equal(got, alone[0]) and torch.equal(k_out, alone[1]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("style", ["blocks", "alternating"])
@pytest.mark.parametrize("size", [(1, 8, 1, 128, 128, 128), (6, 8, 2, 64, 64, 32), (7, 6, 3, 80, 80, 80), (5, 3, 3, 72, 72, 72), (9, 4, 1, 90, 90, 90),
                                  (3, 4, 2, 192, 128, 64), (2, 2, 1, 4, 2, 4), (5, 1, 1, 1024, 512, 1024)])
def test_sizes(dev, size, style, kind):
    run(*size, kind, style, norm=True, interleaved=True)
    run(*size, kind, style, axes=2, page=5, layout="heads")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("style", ["blocks", "alternating"])
def test_many(dev, style, interleaved, kind):
    """Launches that fill the chip: two heads a lane group (of four values a piece: four), whose last group has fewer, with padding
    among the tokens."""
    run(1030, 61, 7, 128, 128, 128, kind, style, norm=interleaved, interleaved=interleaved)
    run(1030, 61, 7, 72, 72, 72, kind, style, axes=4, norm=not interleaved, interleaved=interleaved, layout="heads")


@pytest.mark.parametrize("seed", range(60))
def test_random(dev, seed):
    r = random.Random(3000 + seed)
    tokens, hq, hk, dim, width = sizes(r)
    padding = [(r.randrange(tokens), r.choice([-1, -2 ** 31, 2 ** 31 - 1])) for _ in range(r.randint(0, 3))]
    dtype = r.choice([BF16, F16])
    kw = dict(kind=r.choice(KINDS), style=r.choice(["blocks", "alternating"]), axes=r.randint(1, 4), page=r.choice([1, 3, 16, 64]),
              layout=r.choice(["tokens", "heads"]), norm=r.random() < 0.5, dtype=dtype, table_dtype=r.choice([F32, dtype]), interleaved=r.random() < 0.5,
              index=r.choice([torch.int32, torch.int64]), padding=padding)
    dim_v = r.choice([dim, 2 * r.randint(1, 130)])
    print(tokens, hq, hk, dim, dim_v, width, kw, flush=True)
    run(tokens, hq, hk, dim, dim_v, width, seed=seed, **kw)


def test_captured(dev):
    """A captured append whose positions and slots change between its replays; a token behind the last one is padding."""
    g = torch.Generator().manual_seed(31)
    tokens, hq, hk, dim, total = 5, 8, 2, 128, 64
    turn = dict(cos_sin=table(300, dim).cuda(), sections=[24, 20, 20], alternating=True, interleaved=False)
    qkv, positions = torch.zeros(tokens, hq + 2 * hk, dim, device=dev, dtype=BF16), torch.zeros(3, tokens, device=dev, dtype=torch.int64)
    slots, q_out = torch.full((tokens,), -1, device=dev), torch.empty(tokens, hq, dim, device=dev, dtype=BF16)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    caches = [make_cache(g, "int8_rows", total // 16, 16, (hk, dim), BF16) for _ in range(2)]
    eager = [tuple(t.clone() for t in pair) for pair in caches]

    def put(to, out):
        append_kv(k, v, to[0][0], to[1][0], slots, k_scale=to[0][1], v_scale=to[1][1], q=q, positions=positions, q_out=out, **turn)

    put(caches, q_out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        put(caches, q_out)
    for _ in range(4):
        qkv.copy_(heads(g, tokens, hq + 2 * hk, dim, dtype=BF16))
        positions.copy_(torch.randint(0, 300, (3, tokens), generator=g))
        slots.copy_(make_slots(g, tokens, total // 16, 16, ((4, -1),)))
        graph.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(q_out)
        put(eager, want)
        assert torch.equal(q_out, want)
        for now, ref in zip(caches, eager):
            assert torch.equal(now[0], ref[0]) and torch.equal(now[1], ref[1])
