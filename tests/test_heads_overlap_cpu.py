"""Which memory the operators on heads take for shared: every layout of pages in which the tensors lie apart is served, and one value in
common is refused.  Tensors on the CPU get as far as the check behind it, which asks for CUDA tensors."""
import random

import pytest
import torch

from sglang_amd import append_kv, append_latent, gather_kv, gather_latent, rotate_qk

BF16, F8, F32 = torch.bfloat16, torch.float8_e4m3fn, torch.float32
T, PAGES, PAGE, H, D = 3, 5, 4, 2, 64
KV = torch.zeros(T, H, D, dtype=BF16)
SLOTS = torch.arange(T)


def padded(slot, padding, dtype=BF16):
    """Pages of PAGE slots of `slot` elements, something else behind each page: [pages, PAGE, slot]."""
    return torch.zeros(PAGES, PAGE * slot + padding, dtype=dtype)[:, :PAGE * slot].view(PAGES, PAGE, slot)


def part(slots, first, heads=H, dim=D):
    return slots[..., first:first + heads * dim].view(*slots.shape[:-1], heads, dim)


# (page's padding: one that the slot's size divides, ones that it does not, and that the parts' sizes do not)
@pytest.mark.parametrize("padding", [0, 64, 256, 2, 38, 1000])
def test_keys_and_values_side_by_side_in_padded_pages(padding):
    slots = padded(2 * H * D, padding)
    with pytest.raises(RuntimeError, match="CUDA"):
        append_kv(KV, KV, part(slots, 0), part(slots, H * D), SLOTS)
    with pytest.raises(RuntimeError, match="CUDA"):
        append_kv(KV, KV, part(slots, H * D), part(slots, 0), SLOTS)
    for first in (H * D - 1, 1):
        with pytest.raises(RuntimeError, match="v_cache must not overlap k_cache"):
            append_kv(KV, KV, part(slots, 0), part(slots, first), SLOTS)


@pytest.mark.parametrize("padding", [0, 16, 130, 1000])
def test_heads_side_by_side_in_padded_pages(padding):
    """Keys and values of each head beside each other, pages of heads: [pages, heads, PAGE, (k, v)]."""
    pages = torch.zeros(PAGES, H * PAGE * 2 * D + padding, dtype=BF16)[:, :H * PAGE * 2 * D].view(PAGES, H, PAGE, 2 * D).transpose(1, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        append_kv(KV, KV, pages[..., :D], pages[..., D:], SLOTS)
    with pytest.raises(RuntimeError, match="v_cache must not overlap k_cache"):
        append_kv(KV, KV, pages[..., :D], pages[..., D - 1:-1], SLOTS)


@pytest.mark.parametrize("padding", [0, 4, 60, 1000])
def test_codes_and_scales_in_padded_pages(padding):
    """A slot as bytes: the keys' codes, the values', the scales of both; and scales behind the codes of a whole page."""
    rows = H * D
    raw = padded(2 * rows + 8 * H, padding, torch.uint8)
    k, v = part(raw.view(F8), 0), part(raw.view(F8), rows)
    k_scale, v_scale = (raw[..., 2 * rows + 4 * H * i:2 * rows + 4 * H * (i + 1)].view(F32) for i in range(2))
    with pytest.raises(RuntimeError, match="CUDA"):
        append_kv(KV, KV, k, v, SLOTS, k_scale=k_scale, v_scale=v_scale)
    with pytest.raises(RuntimeError, match="k_scale must not overlap k_cache|v_cache must not overlap k_scale"):
        append_kv(KV, KV, k, v, SLOTS, k_scale=raw[..., 2 * rows - 4:2 * rows - 4 + 4 * H].view(F32), v_scale=v_scale)
    whole = torch.zeros(PAGES, PAGE * (2 * rows + 8 * H) + padding, dtype=torch.uint8)
    codes = whole[:, :2 * PAGE * rows].view(F8).view(PAGES, PAGE, 2, H, D)
    scales = whole[:, 2 * PAGE * rows:2 * PAGE * (rows + 4 * H)].view(F32).view(PAGES, PAGE, 2, H)
    with pytest.raises(RuntimeError, match="CUDA"):
        append_kv(KV, KV, codes[:, :, 0], codes[:, :, 1], SLOTS, k_scale=scales[:, :, 0], v_scale=scales[:, :, 1])
    shifted = whole[:, 2 * PAGE * rows - 4:2 * PAGE * (rows + 4 * H) - 4].view(F32).view(PAGES, PAGE, 2, H)
    with pytest.raises(RuntimeError, match="must not overlap"):
        append_kv(KV, KV, codes[:, :, 0], codes[:, :, 1], SLOTS, k_scale=shifted[:, :, 0], v_scale=scales[:, :, 1])


@pytest.mark.parametrize("padding", [0, 2, 64, 1000])
def test_latent_rows_in_padded_pages(padding):
    slots = padded(576, padding)
    latent, rope, cos_sin = torch.zeros(T, 512, dtype=BF16), torch.zeros(T, 64, dtype=BF16), torch.zeros(9, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        append_latent(latent, rope, slots[..., :512], slots[..., 512:], SLOTS, SLOTS, cos_sin)
    with pytest.raises(RuntimeError, match="rope_cache must not overlap latent_cache"):
        append_latent(latent, rope, slots[..., :512], slots[..., 511:575], SLOTS, SLOTS, cos_sin)


def test_gathered_rows_between_the_slots_of_padded_pages():
    """Outputs in memory that the caches' pages leave free, and in memory that they do not."""
    base = torch.zeros(PAGES, PAGE * 2 * H * D + 2 * H * D + 6, dtype=BF16)
    slots = base[:, :PAGE * 2 * H * D].view(PAGES, PAGE, 2 * H * D)
    free = base[:T, PAGE * 2 * H * D:PAGE * 2 * H * D + H * D].view(T, H, D)
    with pytest.raises(RuntimeError, match="CUDA"):
        gather_kv(part(slots, 0), part(slots, H * D), SLOTS, BF16, k_out=free)
    with pytest.raises(RuntimeError, match="k_out must not overlap v_cache"):
        gather_kv(part(slots, 0), part(slots, H * D), SLOTS, BF16, k_out=base[:T, PAGE * 2 * H * D - 1:PAGE * 2 * H * D - 1 + H * D].view(T, H, D))
    rows = padded(576, 700)
    with pytest.raises(RuntimeError, match="out must not overlap latent_cache"):
        gather_latent(rows[..., :512], rows[..., 512:], SLOTS, BF16, out=rows[0, :T])


@pytest.mark.parametrize("seed", range(300))
def test_random_views_of_one_buffer(seed):
    """Two outputs anywhere in one buffer, against the sets of their elements."""
    r = random.Random(seed)
    tokens = r.choice([1, 2, 3, 7])
    buffer = torch.zeros(4000, dtype=BF16)

    def view():
        heads, dim = r.choice([1, 1, 2, 3]), r.choice([2, 4, 6, 16])
        inner = [dim + r.choice([0, 0, 2, 5, 20])] if r.random() < 0.5 else [0]
        if inner[0]:  # heads inside a token
            step = inner[0]
            token = (heads - 1) * step + dim + r.choice([0, 0, 3, 10, 40])
        else:  # tokens inside a head
            token = dim + r.choice([0, 0, 2, 7, 30])
            step = (tokens - 1) * token + dim + r.choice([0, 1, 25])
        return (tokens, heads, dim), (token, step, 1)

    (q_size, q_step), (k_size, k_step) = view(), view()
    if r.random() < 0.6:  # side by side more often than not
        k_size, k_step = q_size, q_step
    q_at, k_at = r.randrange(60), r.randrange(60)
    q_out, k_out = buffer.as_strided(q_size, q_step, q_at), buffer.as_strided(k_size, k_step, k_at)
    numbers = torch.arange(4000)
    shared = set(numbers.as_strided(q_size, q_step, q_at).flatten().tolist()) & set(numbers.as_strided(k_size, k_step, k_at).flatten().tolist())
    with pytest.raises(RuntimeError, match="k_out must not overlap q_out" if shared else "CUDA"):
        rotate_qk(torch.zeros(q_size, dtype=BF16), torch.zeros(k_size, dtype=BF16), torch.arange(tokens), torch.zeros(10, 2), q_out=q_out, k_out=k_out)


def test_pages_by_the_hundred_thousand():
    """Sizes alone count: the memory is not touched, and the answer does not look at page after page."""
    pages, scale, kv = 1 << 17, torch.zeros(1), torch.zeros(T, 1, 128, dtype=BF16)
    memory = torch.empty(pages * 1088, dtype=torch.uint8)
    k, v, shared = (memory.as_strided((pages, PAGE, 1, 128), (1088, 256, 128, 1), at).view(F8) for at in (0, 128, 127))
    with pytest.raises(RuntimeError, match="CUDA"):
        append_kv(kv, kv, k, v, SLOTS, k_scale=scale, v_scale=scale)
    with pytest.raises(RuntimeError, match="v_cache must not overlap k_cache"):
        append_kv(kv, kv, k, shared, SLOTS, k_scale=scale, v_scale=scale)
