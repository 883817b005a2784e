"""Seeded random sizes, types, axes, caches and layouts of the operators on heads, against their definitions in 64 bits."""
import random

import pytest
import torch

from tests.test_kv_cache_gpu import BF16, F16, KINDS, run_append
from tests.test_rotary_gpu import run

pytestmark = pytest.mark.gpu

F32 = torch.float32


def sizes(r):
    dim = 2 * r.choice([r.randint(1, 64), r.randint(1, 512), 8 * r.randint(1, 64), 4 * r.randint(1, 128), 64])
    width = 2 * r.choice([dim // 2, r.randint(1, dim // 2), min(dim // 2, 32), max(dim // 4, 1)])
    hk = r.randint(1, 9)
    heads = hk * r.choice([1, 1, 2, 3, 8])
    tokens = max(1, min(r.choice([1, 2, r.randint(1, 40), r.randint(1, 700)]), 4_000_000 // (heads * dim)))
    return tokens, heads, hk, dim, width


@pytest.mark.parametrize("seed", range(60))
def test_heads(dev, seed):
    r = random.Random(seed)
    dtype = r.choice([BF16, F16])
    args = sizes(r) + (r.random() < 0.5, r.choice(["one", "blocks", "alternating"]), dtype, r.choice([F32, F32, dtype]),
                       r.choice([torch.int32, torch.int64]), r.choice([None, F32, dtype]))
    print(args, flush=True)
    run(*args, seed=seed)


@pytest.mark.parametrize("seed", range(80))
def test_appends(dev, seed):
    r = random.Random(1000 + seed)
    tokens, hq, hk, dim, width = sizes(r)
    dim_v = r.choice([dim, dim, 2 * r.randint(1, 130)])
    padding = [(r.randrange(tokens), r.choice([-1, -2 ** 31, 2 ** 31 - 1])) for _ in range(r.randint(0, 3))]
    kw = dict(kind=r.choice(KINDS), page=r.choice([1, 3, 16, 64]), layout=r.choice(["tokens", "heads"]), norm=r.random() < 0.5,
              dtype=r.choice([BF16, F16]), interleaved=r.random() < 0.5, index=r.choice([torch.int32, torch.int64]), padding=padding)
    print(tokens, hq, hk, dim, dim_v, width, kw, flush=True)
    run_append(tokens, hq, hk, dim, dim_v, width, seed=seed, **kw)
