"""Caches whose pages hold more than their rows: keys beside values, scales beside codes, something else behind the last slot."""
import pytest
import torch

from sglang_amd import append_kv, append_latent, gather_kv, gather_latent
from tests.head_rows import heads, table
from tests.test_kv_cache_gpu import BF16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("padding", [0, 64, 1000])
def test_keys_and_values_side_by_side_in_padded_pages(dev, padding):
    """A slot as bytes, its keys' codes, its values' and the scales of both, in pages with something else behind the last slot: the same
    bytes as in caches of their own."""
    g = torch.Generator().manual_seed(40)
    tokens, h, dim, pages, page = 21, 2, 64, 5, 8
    rows = h * dim
    slot = 2 * rows + 8 * h
    raw = torch.randint(0, 100, (pages, page * slot + padding), generator=g, dtype=torch.uint8).cuda()
    before = raw.clone()
    inside = raw[:, :page * slot].view(pages, page, slot)
    codes = [inside[..., rows * i:rows * (i + 1)].view(pages, page, h, dim).view(torch.int8) for i in range(2)]
    scales = [inside[..., 2 * rows + 4 * h * i:2 * rows + 4 * h * (i + 1)].view(torch.float32) for i in range(2)]
    k, v = (heads(g, tokens, h, dim, dtype=BF16).cuda() for _ in range(2))
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[3] = -1
    slots = slots.cuda()
    append_kv(k, v, codes[0], codes[1], slots, k_scale=scales[0], v_scale=scales[1])
    own = [(torch.zeros(pages, page, h, dim, device=dev, dtype=torch.int8), torch.zeros(pages, page, h, device=dev)) for _ in range(2)]
    append_kv(k, v, own[0][0], own[1][0], slots, k_scale=own[0][1], v_scale=own[1][1])
    put = slots[slots >= 0]
    at = (put // page, put % page)
    for i in range(2):
        assert torch.equal(codes[i][at], own[i][0][at]) and torch.equal(scales[i][at], own[i][1][at])
    rest = torch.ones(pages, page, dtype=torch.bool, device=dev)
    rest[at] = False
    old = before[:, :page * slot].view(pages, page, slot)
    assert torch.equal(inside[rest], old[rest]) and torch.equal(raw[:, page * slot:], before[:, page * slot:])
    for got, want in zip(gather_kv(codes[0], codes[1], put, BF16, k_scale=scales[0], v_scale=scales[1]),
                         gather_kv(own[0][0], own[1][0], put, BF16, k_scale=own[0][1], v_scale=own[1][1])):
        assert torch.equal(got, want)


def test_latent_rows_in_padded_pages(dev):
    g = torch.Generator().manual_seed(41)
    tokens, pages, page = 20, 4, 16
    base = torch.ones(pages, page * 576 + 200, device=dev, dtype=BF16)
    rows = base[:, :page * 576].view(pages, page, 576)
    latent, rope = heads(g, tokens, 512, dtype=BF16).cuda(), heads(g, tokens, 64, dtype=BF16).cuda()
    slots, positions, cos_sin = torch.randperm(pages * page, generator=g)[:tokens].cuda(), torch.arange(tokens, device=dev), table(32, 64).cuda()
    append_latent(latent, rope, rows[..., :512], rows[..., 512:], slots, positions, cos_sin)
    own = torch.ones(pages, page, 576, device=dev, dtype=BF16)
    append_latent(latent, rope, own[..., :512], own[..., 512:], slots, positions, cos_sin)
    assert torch.equal(rows, own) and (base[:, page * 576:] == 1).all()
    assert torch.equal(gather_latent(rows[..., :512], rows[..., 512:], slots, BF16), gather_latent(own[..., :512], own[..., 512:], slots, BF16))
