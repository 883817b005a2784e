"""Launches of many gathered rows, memory beyond 32-bit offsets, tables at their limit, codes of one slot written twice."""
import pytest
import torch

from sglang_amd import append_kv, gather_kv, gather_latent, rotate_qk
from tests.head_rows import F8, check_16, check_8, heads, normed, table, turned
from tests.test_kv_cache_gpu import BF16, F16, KINDS, bits, gathered, make_cache

pytestmark = pytest.mark.gpu


def enough_rows(units_per_row):
    """Rows enough for four units a lane, whose last workgroup is not full in either part."""
    least = torch.cuda.get_device_properties(0).multi_processor_count * 16384 // units_per_row + 1
    return next(n for n in range(least, least + 1024) if n * units_per_row // 2 % 1024)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,piece", [(128, 8), (72, 8), (36, 4), (90, 1)])
def test_gather_many(dev, dim, piece, kind, dtype):
    """Launches of four units a lane in pieces of eight values, of four and of one."""
    g = torch.Generator().manual_seed(42 + dim)
    h = 7
    rows = enough_rows(2 * h * dim // piece)
    caches = [make_cache(g, kind, 100, 16, (h, dim), dtype) for _ in range(2)]
    slots = torch.randint(-1, 1601, (rows,), generator=g).cuda()
    got = gather_kv(caches[0][0], caches[1][0], slots, dtype, k_scale=caches[0][1], v_scale=caches[1][1])
    for back, (cache, scale) in zip(got, caches):
        assert torch.equal(back.cpu(), gathered(cache, scale, slots, dtype, 1600, (h, dim)))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kind", ["16", "e4m3", "e4m3_groups", "int8_groups"])
def test_gather_many_latents(dev, kind, dtype):
    g = torch.Generator().manual_seed(43)
    rows, c, r = enough_rows(72) + 1, 512, 64
    cache, scale = make_cache(g, kind, 200, 16, (c,), dtype)
    rope_cache, rope_scale = make_cache(g, kind if kind in ("16", "e4m3") else "16", 200, 16, (r,), dtype)
    group = None
    if kind.endswith("_groups"):
        group, scale = 128, torch.rand(200, 16, c // 128, generator=g).cuda()
    slots = torch.randint(-1, 3201, (rows,), generator=g).cuda()
    got = gather_latent(cache, rope_cache, slots, dtype, scale=scale, rope_scale=rope_scale)
    assert torch.equal(got[:, :c].cpu(), gathered(cache, scale, slots, dtype, 3200, (c,), group))
    assert torch.equal(got[:, c:].cpu(), gathered(rope_cache, rope_scale, slots, dtype, 3200, (r,)))


def test_scales_beyond_32_bits(dev):
    """Slots of 2 x 1024 codes and two scales in one buffer of a little over 4 GiB: the last ones' scales lie beyond 2^32 bytes too."""
    slot, h, dim = 2 * 1024 + 8, 2, 1024
    count = (1 << 32) // slot + 100
    raw = torch.zeros(count, slot, device=dev, dtype=torch.uint8)
    cache, scale = raw[:, :h * dim].view(count, h, dim).view(torch.int8), raw[:, h * dim:].view(torch.float32)
    small, small_scale = torch.zeros(count, 1, 2, device=dev, dtype=torch.int8), torch.zeros(count, 1, device=dev)
    g = torch.Generator().manual_seed(44)
    k, v = heads(g, 3, h, dim, dtype=BF16).cuda(), heads(g, 3, 1, 2, dtype=BF16).cuda()
    slots = torch.tensor([count - 1, 5, count - 50], device=dev)
    append_kv(k, v, cache, small, slots, k_scale=scale, v_scale=small_scale)
    assert raw.count_nonzero(dim=1).nonzero().view(-1).tolist() == sorted(slots.tolist())
    check_8(cache[slots].cpu(), *normed(k, None, 1e-6), scales=scale[slots].unsqueeze(-1))
    back, _ = gather_kv(cache, small, slots, BF16, k_scale=scale, v_scale=small_scale)
    assert torch.equal(back, (cache[slots].float() * scale[slots].unsqueeze(-1)).to(BF16))


@pytest.mark.parametrize("axes", [1, 2])
@pytest.mark.parametrize("width,dtype,table_dtype", [(1024, BF16, torch.float32), (128, F16, F16), (6, BF16, torch.float32)])
def test_tables_of_2_gib(dev, width, dtype, table_dtype, axes):
    """The last positions of the longest tables that are served; rows that no position names are left as they were allocated."""
    g = torch.Generator().manual_seed(45)
    count = (1 << 31) // (width * table_dtype.itemsize)
    cos_sin = torch.empty(count, width, device=dev, dtype=table_dtype)
    named = [0, 5, count // 2, count - 2, count - 1]
    rows = table(5, width, table_dtype)
    cos_sin[torch.tensor(named, device=dev)] = rows.cuda()
    choice = torch.randint(-1, 6, (axes, 40), generator=g)  # (-1 and 5: outside)
    choice[:, :5] = 4
    positions = torch.tensor([-1] + named + [count])[choice + 1]
    x = heads(g, 40, 3, width, dtype=dtype).cuda()
    turn = dict(interleaved=False) if axes == 1 else dict(interleaved=False, sections=[width // 2 - width // 4, width // 4], alternating=True)
    if axes == 1:
        choice, positions = choice[0], positions[0]
    got, _ = rotate_qk(x, None, positions.cuda(), cos_sin, **turn)
    check_16(got, *turned(*normed(x, None, 1e-6), choice, rows, **turn))


def test_codes_of_the_same_slot_twice(dev):
    """Every byte of the row is that of one of the two tokens, and so is the scale; all other rows are as they were."""
    g = torch.Generator().manual_seed(46)
    for dim in (128, 72, 90):
        k = heads(g, 3, 2, dim, dtype=BF16).cuda()
        caches = [(torch.zeros(6, 2, dim, device=dev, dtype=F8), torch.zeros(6, 2, device=dev)) for _ in range(2)]
        append_kv(k, k, caches[0][0], caches[1][0], torch.tensor([4, 1, 4], device=dev), k_scale=caches[0][1], v_scale=caches[1][1])
        apart = [(torch.zeros(6, 2, dim, device=dev, dtype=F8), torch.zeros(6, 2, device=dev)) for _ in range(2)]
        append_kv(k, k, apart[0][0], apart[1][0], torch.tensor([0, 1, 2], device=dev), k_scale=apart[0][1], v_scale=apart[1][1])
        for (codes, scale), (one, its) in zip(caches, apart):
            codes, one = bits(codes), bits(one)
            assert ((codes[4] == one[0]) | (codes[4] == one[2])).all() and ((scale[4] == its[0]) | (scale[4] == its[2])).all()
            assert torch.equal(codes[1], one[1]) and torch.equal(scale[1], its[1])
            assert not codes[[0, 2, 3, 5]].any() and not scale[[0, 2, 3, 5]].any()
