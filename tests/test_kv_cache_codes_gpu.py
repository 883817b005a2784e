"""The codes of cached rows bit for bit: what the contract multiplies by, rounded to float32, also next to ties, where a division may
come out on the other side."""
import pytest
import torch

from sglang_amd import append_kv
from tests.head_rows import F8, heads
from tests.test_kv_cache_gpu import BF16, F16, bits

pytestmark = pytest.mark.gpu


def e4m3(y, scale):
    """IEEE arithmetic in 32 bits on the CPU."""
    return (y * torch.where(scale == 0, torch.zeros_like(scale), 1.0 / scale)).clamp(-448.0, 448.0).to(F8)


def rows_with_ties(g, tokens, h, dim, dtype):
    """Rows whose largest value is a power of two times 1.75, as 448 is: every value lies on a code, on a tie or between."""
    x = heads(g, tokens, h, dim, dtype=dtype).float().clamp(-6.9, 6.9)
    x[:, :, 3] = 7.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [128, 72, 90])
@pytest.mark.parametrize("ties", [False, True])
def test_rows(dev, ties, dim, dtype):
    g = torch.Generator().manual_seed(50 + dim)
    tokens, h = 40, 3
    x = rows_with_ties(g, tokens, h, dim, dtype) if ties else heads(g, tokens, h, dim, dtype=dtype)
    x[7, 1] = 0
    peak = x.float().abs().amax(dim=-1)
    slots = torch.arange(tokens, device=dev)
    for kind in (F8, torch.int8):
        caches = [(torch.zeros(tokens, h, dim, device=dev, dtype=kind), torch.full((tokens, h), 5.0, device=dev)) for _ in range(2)]
        append_kv(x.cuda(), x.cuda(), caches[0][0], caches[1][0], slots, k_scale=caches[0][1], v_scale=caches[1][1])
        if kind == F8:
            scale = peak / torch.tensor(448.0)
            codes = e4m3(x.float(), scale.unsqueeze(-1))
        else:
            m = peak.clamp_min(1e-10)
            scale, by = m / torch.tensor(127.0), (torch.tensor(127.0) / m).unsqueeze(-1)
            v = x.float() * by
            codes = (torch.sign(v) * torch.floor(v.abs() + 0.5)).to(torch.int8)
        for cache, found in caches:
            assert torch.equal(found.cpu(), scale) and torch.equal(bits(cache).cpu(), bits(codes))


@pytest.mark.parametrize("dim", [128, 72, 90])
def test_given_scales(dev, dim):
    """Ones that ties hang on, one that is zero: its codes are zeros."""
    g = torch.Generator().manual_seed(60 + dim)
    tokens, h = 40, 4
    x = rows_with_ties(g, tokens, h, dim, BF16)
    scale = torch.tensor([7.0 / 448.0, 0.0213, 0.0, 3.0])
    caches = [torch.full((tokens, h, dim), 1.0, device=dev).to(F8) for _ in range(2)]
    append_kv(x.cuda(), x.cuda(), caches[0], caches[1], torch.arange(tokens, device=dev), k_scale=scale.cuda(), v_scale=scale[:1].cuda())
    assert torch.equal(bits(caches[0]).cpu(), bits(e4m3(x.float(), scale.view(-1, 1)))) and not caches[0][:, 2].float().any()
    assert torch.equal(bits(caches[1]).cpu(), bits(e4m3(x.float(), scale[:1].view(-1, 1))))
