"""What rotations of heads, appends and gathers refuse, before any launch: tensors on the CPU get as far as the checks."""
import ctypes

import pytest
import torch

from sglang_amd import append_kv, append_latent, gather_kv, gather_latent, norm_rotate_qk, rotate_qk
from sglang_amd._lib import lib

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn
T = 6


def Z(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def rotate(q=None, k=None, positions=None, cos_sin=None, **kw):
    rotate_qk(Z(T, 4, 64) if q is None else q, Z(T, 2, 64) if k is None else k, torch.arange(T) if positions is None else positions,
              Z(10, 64, dtype=torch.float32) if cos_sin is None else cos_sin, **kw)


_SAME = Z(T, 4, 64)
_ROWS = Z(T, 6, 64)

ROTATE = [
    ("must be a CUDA tensor", dict()),
    ("q must be \\[tokens", dict(q=Z(T, 64))),
    ("Half or BFloat16", dict(q=Z(T, 4, 64, dtype=torch.float32))),
    ("k must have the dtype", dict(k=Z(T, 2, 64, dtype=torch.float16))),
    ("k must have as many tokens", dict(k=Z(T + 1, 2, 64))),
    ("even sizes up to 1024", dict(q=Z(T, 4, 65))),
    ("even sizes up to 1024", dict(q=Z(T, 4, 1026))),
    ("q rows must be contiguous", dict(q=Z(T, 64, 4).transpose(1, 2))),
    ("positions must be \\[tokens\\]", dict(positions=torch.arange(T + 1))),
    ("positions must be \\[tokens\\]", dict(positions=torch.zeros(3, T, dtype=torch.long))),
    ("positions must be Int or Long", dict(positions=torch.zeros(T))),
    ("cos_sin must be \\[positions", dict(cos_sin=Z(64))),
    ("at least one position", dict(cos_sin=Z(0, 64, dtype=torch.float32))),
    ("even, 2 to 1024", dict(cos_sin=Z(10, 63, dtype=torch.float32))),
    ("a rotated width of 66 for q of 64", dict(cos_sin=Z(10, 66, dtype=torch.float32))),
    ("cos_sin must be Float32", dict(cos_sin=Z(10, 64, dtype=torch.float16))),
    ("cos_sin rows must be contiguous", dict(cos_sin=Z(64, 10, dtype=torch.float32).t())),
    ("must add up to the 32", dict(positions=torch.zeros(2, T, dtype=torch.long), sections=[16, 15])),
    ("must not be negative", dict(positions=torch.zeros(2, T, dtype=torch.long), sections=[33, -1])),
    ("positions must be \\[axes", dict(positions=torch.zeros(3, T, dtype=torch.long), sections=[16, 16])),
    ("one to four axes", dict(positions=torch.zeros(5, T, dtype=torch.long), sections=[8, 8, 8, 4, 4])),
    ("axis 1 has no 17 turns", dict(positions=torch.zeros(2, T, dtype=torch.long), sections=[15, 17], alternating=True)),
    ("need their sections", dict(alternating=True)),
    ("q_out must match", dict(q_out=Z(T, 4, 62))),
    ("q_out must match", dict(q_out=Z(T, 4, 64, dtype=torch.float16))),
    ("q_out must not be expanded", dict(q_out=Z(1, 4, 64).expand(T, 4, 64))),
    ("q_out rows must be contiguous", dict(q_out=Z(T, 64, 4).transpose(1, 2))),
    ("k_out must not overlap q", dict(q=_ROWS[:, :4], k=_ROWS[:, 4:], k_out=_ROWS[:, 3:5])),
    ("q_out must not overlap q", dict(q=_SAME, q_out=_SAME.view(-1).view(4, T, 64).transpose(0, 1))),
]


@pytest.mark.parametrize("text,kw", ROTATE, ids=range(len(ROTATE)))
def test_rotations(text, kw):
    with pytest.raises(RuntimeError, match=text):
        rotate(**kw)


def test_a_single_tensor_has_no_second_output():
    with pytest.raises(RuntimeError, match="k_out goes with k"):
        rotate_qk(Z(T, 4, 64), None, torch.arange(T), Z(10, 64, dtype=torch.float32), k_out=Z(T, 4, 64))


def test_views_of_one_projection_are_no_overlap():
    """q and k in place in one buffer, interleaved by tokens or by heads: refused for being on the CPU only."""
    for rows in (_ROWS, Z(1, 6, 64), Z(6, T, 64).transpose(0, 1)):
        n = rows.shape[0]
        with pytest.raises(RuntimeError, match="CUDA"):
            rotate_qk(rows[:, :4], rows[:, 4:], torch.arange(n), Z(10, 64, dtype=torch.float32), q_out=rows[:, :4], k_out=rows[:, 4:])
    wide = Z(T, 3, 128)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotate_qk(wide[..., :64], wide[..., 64:], torch.arange(T), Z(10, 64, dtype=torch.float32), q_out=wide[..., :64], k_out=wide[..., 64:])
    with pytest.raises(RuntimeError, match="q_out must not overlap q"):
        rotate_qk(wide[..., :64], wide[..., 64:], torch.arange(T), Z(10, 64, dtype=torch.float32), q_out=wide[..., 60:124])


def test_norms():
    cos_sin = Z(10, 64, dtype=torch.float32)
    good = Z(64)
    for text, w, eps in (("q_weight must be contiguous", Z(63), 1e-6), ("q_weight must be contiguous", Z(64, 1), 1e-6),
                         ("q_weight must be Float32", Z(64, dtype=torch.float16), 1e-6), ("epsilon", good, -1.0), ("epsilon", good, float("nan")),
                         ("epsilon", good, float("inf")), ("CUDA", good, 0.0)):
        with pytest.raises(RuntimeError, match=text):
            norm_rotate_qk(Z(T, 4, 64), Z(T, 2, 64), w, good, eps, torch.arange(T), cos_sin)


def append(kind=BF16, **kw):
    args = dict(k=Z(T, 2, 64), v=Z(T, 2, 64), k_cache=Z(5, 4, 2, 64, dtype=kind), v_cache=Z(5, 4, 2, 64, dtype=kind), slots=torch.arange(T))
    args.update(kw)
    append_kv(**args)


F32 = torch.float32
_KV = Z(5, 4, 2, 64)

APPEND = [
    ("CUDA", dict()),
    ("CUDA", dict(kind=F8, k_scale=Z(1, dtype=F32), v_scale=Z(5, 4, 2, dtype=F32))),
    ("CUDA", dict(kind=torch.int8, k_scale=Z(5, 4, 2, dtype=F32), v_scale=Z(5, 4, 2, dtype=F32))),
    ("k_scale is needed", dict(kind=F8)),
    ("k_scale goes with 8-bit", dict(k_scale=Z(1, dtype=F32))),
    ("Char rows have scales", dict(kind=torch.int8, k_scale=Z(1, dtype=F32), v_scale=Z(5, 4, 2, dtype=F32))),
    ("one number, or one per head", dict(kind=F8, k_scale=Z(3, dtype=F32), v_scale=Z(1, dtype=F32))),
    ("k_scale must have the cache's slots", dict(kind=F8, k_scale=Z(5, 3, 2, dtype=F32), v_scale=Z(1, dtype=F32))),
    ("k_scale must be one per head of a row", dict(kind=F8, k_scale=Z(5, 4, 1, dtype=F32), v_scale=Z(1, dtype=F32))),
    ("k_scale must have the cache's slots", dict(kind=F8, k_scale=Z(20, 2, dtype=F32), v_scale=Z(1, dtype=F32))),
    ("k_scale must be Float32", dict(kind=F8, k_scale=Z(1), v_scale=Z(1, dtype=F32))),
    ("must have the dtype of the heads", dict(kind=torch.float16)),
    ("a cache must be", dict(kind=torch.float32)),
    ("slots must be 1D", dict(slots=torch.zeros(T, 1, dtype=torch.long))),
    ("slots must be one per token", dict(slots=torch.arange(T - 1))),
    ("slots must be Int or Long", dict(slots=torch.zeros(T))),
    ("k_cache must be \\[slots", dict(k_cache=Z(5, 64))),
    ("k_cache rows must be \\[2, 64\\]", dict(k_cache=Z(5, 4, 3, 64))),
    ("k_cache rows must be \\[2, 64\\]", dict(k_cache=Z(5, 4, 2, 62))),
    ("k_cache rows must be contiguous", dict(k_cache=Z(5, 4, 64, 2).transpose(2, 3))),
    ("v_cache must have the pages", dict(v_cache=Z(4, 5, 2, 64))),
    ("pages must not be empty", dict(k_cache=Z(5, 0, 2, 64))),
    ("k_cache must not be expanded", dict(k_cache=Z(1, 4, 2, 64).expand(5, 4, 2, 64))),
    ("v_cache must not overlap k_cache", dict(k_cache=_KV, v_cache=_KV)),
    ("k_cache must not overlap k", dict(k=_KV.view(20, 2, 64)[:T], k_cache=_KV)),
    ("v_scale must not overlap k_scale", dict(kind=F8, k_scale=(s := Z(5, 4, 2, dtype=F32)), v_scale=s)),
    ("positions and cos_sin go together", dict(positions=torch.arange(T))),
    ("a rotation needs positions", dict(interleaved=True)),
    ("q is only taken", dict(q=Z(T, 4, 64))),
    ("go with q", dict(q_out=Z(T, 4, 64))),
    ("go with q", dict(q_weight=Z(64))),
    ("k must be \\[tokens", dict(k=Z(T, 64))),
    ("v must have as many tokens", dict(v=Z(T - 1, 2, 64))),
    ("k_out must not overlap v", dict(v=(v := Z(T, 2, 64)), k_out=v)),
    ("a rotated width of 64 for q of 32", dict(q=Z(T, 4, 32), positions=torch.arange(T), cos_sin=Z(9, 64, dtype=F32))),
]


@pytest.mark.parametrize("text,kw", APPEND, ids=range(len(APPEND)))
def test_appends(text, kw):
    with pytest.raises(RuntimeError, match=text):
        append(**kw)


def test_halves_of_one_cache_buffer_are_no_overlap():
    both = Z(5, 2, 4, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        append(k_cache=both[:, 0], v_cache=both[:, 1])
    with pytest.raises(RuntimeError, match="CUDA"):
        append(k_cache=both.transpose(1, 2)[:, :, 0], v_cache=both.transpose(1, 2)[:, :, 1])


def latent(kind=BF16, **kw):
    rows = Z(20, 576, dtype=kind)
    args = dict(latent=Z(T, 512), rope=Z(T, 64), latent_cache=rows[:, :512], rope_cache=rows[:, 512:], slots=torch.arange(T),
                positions=torch.arange(T), cos_sin=Z(10, 64, dtype=F32))
    args.update(kw)
    append_latent(**args)


LATENT = [
    ("CUDA", dict()),
    ("CUDA", dict(kind=F8, scale=Z(1, dtype=F32), rope_scale=Z(1, dtype=F32))),
    ("CUDA", dict(latent_cache=Z(20, 512, dtype=F8), scale=Z(20, 4, dtype=F32))),
    ("one per row, or one per 128", dict(latent_cache=Z(20, 512, dtype=F8), scale=Z(20, 8, dtype=F32))),
    ("one per row, or one per 128", dict(latent=Z(T, 130), latent_cache=Z(20, 130, dtype=F8), scale=Z(20, 2, dtype=F32))),
    ("the rotated part is kept", dict(rope_cache=Z(20, 64, dtype=torch.int8), rope_scale=Z(20, 1, dtype=F32))),
    ("the rotated part is kept", dict(rope_cache=Z(20, 64, dtype=F8), rope_scale=Z(20, 1, dtype=F32))),
    ("rope_scale is needed", dict(rope_cache=Z(20, 64, dtype=F8))),
    ("latent and rope must be", dict(rope=Z(T + 1, 64))),
    ("both the same", dict(rope=Z(T, 64, dtype=torch.float16))),
    ("q_out goes with q_rope", dict(q_out=Z(T, 4, 64))),
    ("a rotated width of 64 for rope of 32", dict(rope=Z(T, 32), rope_cache=Z(20, 32))),
    ("rope_cache must have the pages", dict(rope_cache=Z(21, 64))),
    ("rope_cache must not overlap latent_cache", dict(latent_cache=(c := Z(20, 576))[:, :512], rope_cache=c[:, 500:564])),
    ("weight must be contiguous", dict(weight=Z(64))),
]


@pytest.mark.parametrize("text,kw", LATENT, ids=range(len(LATENT)))
def test_latents(text, kw):
    with pytest.raises(RuntimeError, match=text):
        latent(**kw)


def test_gathers():
    cache, codes, slots = Z(5, 4, 2, 64), Z(5, 4, 2, 64, dtype=F8), torch.arange(3)
    scale = Z(5, 4, 2, dtype=F32)
    for text, args, kw in (
            ("CUDA", (cache, cache, slots, BF16), {}),
            ("CUDA", (codes, codes, slots, torch.float16), dict(k_scale=scale, v_scale=scale)),
            ("dtype must be", (cache, cache, slots, torch.float32), {}),
            ("must have the dtype of the heads", (cache, cache, slots, torch.float16), {}),
            ("k_scale is needed", (codes, codes, slots, BF16), {}),
            ("must have the pages", (cache, Z(4, 5, 2, 64), slots, BF16), {}),
            ("up to 1024", (Z(5, 4, 2, 1025), cache, slots, BF16), {}),
            ("k_out must be", (cache, cache, slots, BF16), dict(k_out=Z(3, 2, 62))),
            ("k_out must not overlap k_cache", (cache, Z(5, 4, 2, 64), slots, BF16), dict(k_out=cache.view(20, 2, 64)[:3])),
            ("v_out must not overlap k_out", (cache, cache, slots, BF16), dict(k_out=(o := Z(3, 2, 64)), v_out=o)),
            ("k_out must not be expanded", (cache, cache, slots, BF16), dict(k_out=Z(1, 2, 64).expand(3, 2, 64)))):
        with pytest.raises(RuntimeError, match=text):
            gather_kv(*args, **kw)
    with pytest.raises(RuntimeError, match="out must be \\[rows, 576\\]"):
        gather_latent(Z(20, 512), Z(20, 64), slots, BF16, out=Z(3, 575))
    with pytest.raises(RuntimeError, match="out rows must be contiguous"):
        gather_latent(Z(20, 512), Z(20, 64), slots, BF16, out=Z(576, 3).t())


class Slots(ctypes.Structure):
    _fields_ = [("slots", ctypes.c_void_p), ("slots_dtype", ctypes.c_int), ("slot_stride", ctypes.c_int64), ("page_size", ctypes.c_int64),
                ("pages", ctypes.c_int64)]


class Rotation(ctypes.Structure):
    _fields_ = [("cos_sin", ctypes.c_void_p), ("table_dtype", ctypes.c_int), ("table_rows", ctypes.c_int64), ("table_stride", ctypes.c_int64),
                ("width", ctypes.c_int64), ("interleaved", ctypes.c_int), ("positions", ctypes.c_void_p), ("positions_dtype", ctypes.c_int),
                ("axis_stride", ctypes.c_int64), ("position_stride", ctypes.c_int64), ("axes", ctypes.c_int), ("sections", ctypes.c_int32 * 4),
                ("alternating", ctypes.c_int)]


class Heads(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("x_token", ctypes.c_int64), ("x_head", ctypes.c_int64), ("heads", ctypes.c_int64), ("dim", ctypes.c_int64),
                ("weight", ctypes.c_void_p), ("weight_dtype", ctypes.c_int), ("eps", ctypes.c_float), ("rotate", ctypes.c_int), ("out", ctypes.c_void_p),
                ("out_token", ctypes.c_int64), ("out_head", ctypes.c_int64), ("cache", ctypes.c_void_p), ("cache_dtype", ctypes.c_int),
                ("cache_page", ctypes.c_int64), ("cache_slot", ctypes.c_int64), ("cache_head", ctypes.c_int64), ("given_scale", ctypes.c_void_p),
                ("given_head", ctypes.c_int64), ("scales", ctypes.c_void_p), ("scales_page", ctypes.c_int64), ("scales_slot", ctypes.c_int64),
                ("scales_head", ctypes.c_int64), ("scales_group", ctypes.c_int64), ("scale_group", ctypes.c_int64)]


def test_c_interface_refuses_before_any_launch():
    """Addresses that are never followed: the sizes and types alone are enough for an error code and its text."""
    def heads(**kw):
        return Heads(**dict(dict(x=4096, x_token=64, x_head=64, heads=1, dim=64, weight_dtype=2, eps=1e-6, out=4096, out_token=64, out_head=64), **kw))

    def slots(**kw):
        return Slots(**dict(dict(slots=4096, slots_dtype=6, slot_stride=1, page_size=16, pages=4), **kw))

    def rotation(**kw):
        return Rotation(**dict(dict(cos_sin=4096, table_dtype=0, table_rows=10, table_stride=64, width=64, positions=4096, positions_dtype=6,
                                    position_stride=1, axes=1), **kw))

    to_cache = dict(out=None, cache=4096, cache_dtype=3, cache_page=1024, cache_slot=64)
    for text, tokens, dtype, part, r, s in (
            (b"Half or BFloat16", 1, 0, heads(), None, None),
            (b"bad token count", -1, 2, heads(), None, None),
            (b"bad token count", 1 << 31, 2, heads(), None, None),
            (b"even sizes up to 1024", 1, 2, heads(dim=65), None, None),
            (b"even sizes up to 1024", 1, 2, heads(dim=2048), None, None),
            (b"null heads", 1, 2, heads(x=None), None, None),
            (b"go nowhere", 1, 2, heads(out=None), None, None),
            (b"negative strides", 1, 2, heads(x_token=-64), None, None),
            (b"without its table", 1, 2, heads(rotate=1), None, None),
            (b"even, 2 to 1024", 1, 2, heads(rotate=1), rotation(width=0), None),
            (b"a rotated width of 128 in heads of 64", 1, 2, heads(rotate=1), rotation(width=128), None),
            (b"a table of 0 positions", 1, 2, heads(rotate=1), rotation(table_rows=0), None),
            (b"one to 2 GiB", 1, 2, heads(rotate=1), rotation(table_rows=(1 << 23) + 1), None),
            (b"one to 2 GiB", 1, 2, heads(rotate=1), rotation(table_dtype=2, table_rows=(1 << 24) + 1), None),
            (b"one to 2 GiB", 1, 2, heads(rotate=1), rotation(table_stride=1 << 40), None),
            (b"one to 2 GiB", 1, 2, heads(rotate=1), rotation(table_rows=(1 << 31) - 1, table_stride=1 << 62), None),
            (b"one to 2 GiB", 1, 2, heads(rotate=1), rotation(table_stride=-64), None),
            (b"null table", 1, 2, heads(rotate=1), rotation(positions=None), None),
            (b"positions must be", 1, 2, heads(rotate=1), rotation(positions_dtype=0), None),
            (b"the table must be", 1, 2, heads(rotate=1), rotation(table_dtype=1), None),
            (b"one to four", 1, 2, heads(rotate=1), rotation(axes=5), None),
            (b"sections of 31 pairs", 1, 2, heads(rotate=1), rotation(axes=2, sections=(ctypes.c_int32 * 4)(16, 15, 0, 0)), None),
            (b"no 17 turns", 1, 2, heads(rotate=1), rotation(axes=2, alternating=1, sections=(ctypes.c_int32 * 4)(15, 17, 0, 0)), None),
            (b"a norm weight must be", 1, 2, heads(weight=4096, weight_dtype=1), None, None),
            (b"epsilon", 1, 2, heads(weight=4096, eps=-1.0), None, None),
            (b"a cache needs slots", 1, 2, heads(**to_cache, scales=4096, scale_group=64), None, None),
            (b"either one given scale or scales", 1, 2, heads(**to_cache), None, slots()),
            (b"either one given scale or scales", 1, 2, heads(**to_cache, scales=4096, given_scale=4096), None, slots()),
            (b"a 16-bit cache has no scales", 1, 2, heads(**dict(to_cache, cache_dtype=2), given_scale=4096), None, slots()),
            (b"a cache is of the activations' type", 1, 2, heads(**dict(to_cache, cache_dtype=1), given_scale=4096), None, slots()),
            (b"Char rows have scales", 1, 2, heads(**dict(to_cache, cache_dtype=4), given_scale=4096), None, slots()),
            (b"per 128 values", 1, 2, heads(**to_cache, scales=4096, scale_group=32), None, slots()),
            (b"slots must be I32 or I64", 1, 2, heads(**to_cache, given_scale=4096), None, slots(slots_dtype=0)),
            (b"2^31 slots", 1, 2, heads(**to_cache, given_scale=4096), None, slots(pages=1 << 30)),
            (b"too many for one launch", (1 << 31) - 1, 2, heads(), None, None)):
        rc = lib.sglamd_head_rows(ctypes.byref(part), 1, tokens, dtype, r and ctypes.byref(r), s and ctypes.byref(s), None)
        assert rc == -1 and text in lib.sglamd_last_error(), (text, rc, lib.sglamd_last_error())
    assert lib.sglamd_head_rows(None, 1, 1, 2, None, None, None) == -1
    assert lib.sglamd_head_rows(ctypes.byref(heads()), 5, 1, 2, None, None, None) == -1
    assert lib.sglamd_head_rows(ctypes.byref(heads()), 1, 0, 2, None, None, None) == 0  # nothing to do
    assert lib.sglamd_gather_head_rows(None, 1, 1, 2, None, None) == -1
