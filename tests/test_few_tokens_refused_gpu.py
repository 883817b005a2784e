"""Sizes that the expert layer of a few tokens refuses: before it asks for memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,topk,i", [(64, 64, 4096), (13, 5, 4096), (65, 1, 4096), (1, 65, 4096), (4, 2, 16400)])
def test_refused_before_any_allocation(dev, m, topk, i):
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens

    h = 16
    t = dict(hidden_q=torch.zeros(m, h, device=dev, dtype=torch.int8), hidden_scale=torch.ones(m, 1, device=dev),
             w1=torch.zeros(1, 2 * i, h, device=dev, dtype=torch.int8), w2=torch.zeros(1, h, i, device=dev, dtype=torch.int8),
             w1_scale=torch.ones(1, 2 * i, 1, device=dev), w2_scale=torch.ones(1, h, 1, device=dev),
             topk_weights=torch.ones(m, topk, device=dev), topk_ids=torch.zeros(m, topk, device=dev, dtype=torch.int32))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(NotImplementedError):
        fused_experts_few_tokens(**t)
    assert torch.cuda.max_memory_allocated() == before
