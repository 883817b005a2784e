"""The expert layer of a few tokens on rows so long that the launches ask for more than 56 KB of LDS: four rows of 16384 or two of
32768 codes in the first, eight waves' rows of 16384 in the second."""
import pytest
import torch

from .test_few_tokens_gpu import _check, _layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("m,e,topk,h,i", [(4, 2, 2, 16384, 32), (2, 2, 1, 32768, 16), (1, 1, 1, 32768, 16), (4, 2, 2, 64, 16384), (1, 8, 8, 64, 16384),
                                          (4, 3, 2, 16384, 32), (3, 1, 1, 32768, 48), (2, 2, 2, 4096, 8208), (8, 2, 1, 4112, 4112)])
def test_layer(dev, int8, m, e, topk, h, i):
    from sglang_amd.moe_runner.few_tokens import fused_experts_few_tokens

    t = _layer(dev, m, e, topk, h, i, int8, m + e + h)
    print(f"few tokens {m} x {topk} of {e}, {h} x {i}, int8 {int8}", flush=True)
    out = fused_experts_few_tokens(**t)
    _check(out, t)
    assert torch.equal(out, fused_experts_few_tokens(**t))
