"""Rotary positions and RMSNorm of heads against their definition in 64 bits."""
import pytest
import torch

from sglang_amd import norm_rotate_qk, rotate_qk
from tests.head_rows import check_16, heads, normed, table, turned

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6

# tokens, query heads, key heads, head size, rotated width: pieces of 8, 4 and 1 values, idle lanes, one lane, all lanes
SIZES = [(1, 1, 1, 2, 2), (1, 64, 8, 128, 128), (3, 5, 1, 64, 64), (7, 4, 2, 64, 32), (33, 3, 3, 80, 80), (5, 6, 2, 80, 40), (9, 2, 1, 72, 72),
         (4, 7, 2, 90, 90), (6, 3, 1, 96, 96), (2, 4, 4, 192, 64), (3, 2, 1, 256, 256), (2, 3, 1, 256, 64), (1, 2, 1, 1024, 1024), (2, 1, 1, 520, 520),
         (2, 1, 1, 1022, 6), (2, 1, 1, 514, 514), (300, 16, 2, 128, 128), (257, 9, 5, 128, 64)]


def run(tokens, hq, hk, dim, width, interleaved, axes, dtype, table_dtype, index_dtype, weight_dtype, seed=0, views=True):
    dev = torch.device("cuda")
    g = torch.Generator().manual_seed(1000 * tokens + dim + seed)
    qkv = heads(g, tokens, hq + 2 * hk, dim, dtype=dtype).to(dev)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    cos_sin = table(500, width, table_dtype).to(dev)
    half = width // 2
    sections = alternating = None
    if axes == "one":
        positions = torch.randint(0, 500, (tokens,), generator=g)
    else:
        count = 3 if half >= 3 else 2 if half == 2 else 1
        third = half // count
        sections = [half - (count - 1) * third] + [third] * (count - 1)
        if axes == "blocks":
            sections = sections[::-1]
        alternating = axes == "alternating"
        positions = torch.randint(0, 500, (count, tokens), generator=g)
        positions[:, ::3] = positions[:1, ::3]  # text: the same on every axis
    positions = positions.to(index_dtype).to(dev)
    turn = dict(interleaved=interleaved, sections=sections, alternating=bool(alternating))
    weights = [None, None]
    if weight_dtype is None:
        got = rotate_qk(q, k, positions, cos_sin, **turn)
    else:
        weights = [(torch.rand(dim, generator=g) + 0.5).to(weight_dtype).to(dev) for _ in range(2)]
        got = norm_rotate_qk(q, k, *weights, EPS, positions, cos_sin, **turn)
    for x, w, out in zip((q, k), weights, got):
        assert out.shape == x.shape and out.dtype == dtype and out.is_contiguous()
        check_16(out, *turned(*normed(x, w, EPS), positions, cos_sin, **turn))


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_sizes(dev, size, interleaved, norm):
    run(*size, interleaved, "one", BF16, F32, torch.int64, BF16 if norm else None)


@pytest.mark.parametrize("axes", ["blocks", "alternating"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_axes(dev, size, interleaved, axes):
    run(*size, interleaved, axes, BF16, F32, torch.int64, BF16 if size[0] % 2 else None)


@pytest.mark.parametrize("weight_dtype", [None, F16, F32])
@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("table_dtype", [F16, F32])
@pytest.mark.parametrize("axes", ["one", "alternating"])
def test_types(dev, axes, table_dtype, index_dtype, weight_dtype):
    for size in ((5, 3, 2, 128, 128), (3, 3, 1, 72, 72), (3, 2, 1, 90, 90)):
        run(*size, False, axes, F16, table_dtype, index_dtype, weight_dtype)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("axes", ["one", "blocks", "alternating"])
def test_many_heads_per_lane_group(dev, axes, interleaved):
    """Launches that fill the chip may take two or four heads of a token at a time; head counts that are no multiple of either."""
    for hq, hk, dim, width in ((61, 7, 128, 128), (64, 2, 128, 64), (61, 7, 72, 72), (64, 2, 80, 40)):
        run(1030, hq, hk, dim, width, interleaved, axes, BF16, F32, torch.int64, BF16)


def test_section_counts(dev):
    """One to four axes, empty sections among them."""
    g = torch.Generator().manual_seed(5)
    x = heads(g, 6, 2, 64, dtype=BF16).to(dev)
    cos_sin = table(100, 64).to(dev)
    for sections, alternating in (([32], False), ([32], True), ([0, 32], False), ([16, 16], True), ([20, 12], True), ([8, 0, 24], False),
                                  ([12, 10, 10], True), ([24, 0, 8], True), ([8, 8, 8, 8], False), ([8, 8, 8, 8], True), ([1, 2, 3, 26], False),
                                  ([29, 1, 1, 1], True)):
        positions = torch.randint(0, 100, (len(sections), 6), generator=g).to(dev)
        for interleaved in (False, True):
            turn = dict(interleaved=interleaved, sections=sections, alternating=alternating)
            out, none = rotate_qk(x, None, positions, cos_sin, **turn)
            assert none is None
            check_16(out, *turned(*normed(x, None, EPS), positions, cos_sin, **turn))


def test_views_offsets_and_in_place(dev):
    """Heads that begin anywhere, rows any distance apart, an output in place, one in a strided buffer."""
    g = torch.Generator().manual_seed(6)
    for dim, width in ((128, 128), (64, 64), (72, 72), (90, 90)):
        buf = heads(g, 9, 5, dim + 3, dtype=BF16).to(dev)
        q, k = buf[:, :3, 1:1 + dim], buf[:, 3:, 2:2 + dim]
        wide = torch.full((9, 2, 2 * dim + 1), 7.0, dtype=BF16, device=dev)
        cos_sin = table(64, width + 6).to(dev)[:, 3:3 + width]
        positions = torch.randint(0, 64, (18,), generator=g).to(dev)[::2]
        want = [turned(*normed(x, None, EPS), positions, cos_sin, False) for x in (q, k)]
        before = buf.clone()
        k_out = wide[:, :, dim:2 * dim]
        got = rotate_qk(q, k, positions, cos_sin, q_out=q, k_out=k_out)
        assert got[0].data_ptr() == q.data_ptr() and got[1].data_ptr() == k_out.data_ptr()
        check_16(got[0], *want[0])
        check_16(got[1], *want[1])
        rest = torch.ones_like(buf, dtype=torch.bool)
        rest[:, :3, 1:1 + dim] = False
        assert torch.equal(buf[rest], before[rest])
        assert (wide[:, :, :dim] == 7).all() and (wide[:, :, 2 * dim:] == 7).all()


def test_transposed_and_repeated_inputs(dev):
    g = torch.Generator().manual_seed(7)
    x = heads(g, 4, 6, 64, dtype=F16).to(dev).transpose(0, 1)  # [6 tokens, 4 heads]
    one = heads(g, 1, 1, 64, dtype=F16).to(dev).expand(6, 3, 64)
    cos_sin, positions = table(50, 64).to(dev), torch.randint(0, 50, (1,), generator=g).to(dev).expand(6)
    q, k = rotate_qk(x, one, positions, cos_sin)
    check_16(q, *turned(*normed(x, None, EPS), positions, cos_sin, False))
    check_16(k, *turned(*normed(one, None, EPS), positions, cos_sin, False))


def test_positions_outside_of_the_table(dev):
    g = torch.Generator().manual_seed(8)
    x = heads(g, 6, 3, 128, dtype=BF16).to(dev)
    cos_sin = table(40, 64).to(dev)
    positions = torch.tensor([39, 40, -1, 0, 2 ** 40, -2 ** 62], device=dev)
    for kind in (positions, positions.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)):
        out, _ = rotate_qk(x, None, kind, cos_sin)
        check_16(out, *turned(*normed(x, None, EPS), kind, cos_sin, False))
        assert torch.isnan(out[1, :, :64]).all() and not torch.isnan(out[:, :, 64:]).any() and not torch.isnan(out[0]).any()
    pos3 = torch.stack([positions, torch.zeros_like(positions), torch.ones_like(positions)])
    for alternating in (False, True):
        turn = dict(sections=[12, 10, 10], alternating=alternating)
        out, _ = rotate_qk(x, None, pos3, cos_sin, **turn)
        check_16(out, *turned(*normed(x, None, EPS), pos3, cos_sin, False, **turn))


def test_extreme_values(dev):
    """A norm of a head of zeros, of tiny and of huge values; NaN and infinity stay in their head."""
    w = torch.ones(64, device=dev)
    x = torch.ones(8, 1, 64, device=dev, dtype=BF16)
    x[0] = 0
    x[1] = 1e-30
    x[2] = 1e18
    x[3] = 1e30  # squares beyond float32
    x[4, 0, 5] = float("inf")
    x[5, 0, 5] = float("nan")
    cos_sin, positions = table(20, 64).to(dev), torch.arange(8, device=dev)
    out, _ = norm_rotate_qk(x, x, w, w, EPS, positions, cos_sin)
    want, off = turned(*normed(x, w, EPS), positions, cos_sin, False)
    for row in (0, 1, 2, 6, 7):
        check_16(out[row:row + 1], want[row:row + 1], off[row:row + 1])
    assert torch.isnan(out[3:6]).all()
    plain, _ = rotate_qk(x, None, positions, cos_sin)
    assert torch.isnan(plain[5, 0, [5, 37]]).all() and torch.isnan(plain).sum() == 2
    assert torch.isfinite(plain[3].float()).all()


def test_no_tokens_and_no_heads(dev):
    cos_sin = table(10, 64).to(dev)
    q, k = torch.empty(0, 4, 64, device=dev, dtype=BF16), torch.empty(0, 1, 64, device=dev, dtype=BF16)
    got = rotate_qk(q, k, torch.empty(0, device=dev, dtype=torch.int64), cos_sin)
    assert got[0].shape == q.shape and got[1].shape == k.shape
    q, k = torch.empty(3, 0, 64, device=dev, dtype=BF16), torch.ones(3, 2, 64, device=dev, dtype=BF16)
    positions = torch.arange(3, device=dev)
    got = rotate_qk(q, k, positions, cos_sin)
    assert got[0].shape == q.shape
    check_16(got[1], *turned(*normed(k, None, EPS), positions, cos_sin, False))


def test_other_stream_and_graph(dev):
    """Captured and replayed with new values and the program's own work between the replays."""
    g = torch.Generator().manual_seed(9)
    q, k = heads(g, 5, 8, 128, dtype=BF16).to(dev), heads(g, 5, 2, 128, dtype=BF16).to(dev)
    w = (torch.rand(128, generator=g) + 0.5).to(dev)
    cos_sin, positions = table(100, 128).to(dev), torch.randint(0, 100, (5,), generator=g).to(dev)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm_rotate_qk(q, k, w, w, EPS, positions, cos_sin, q_out=q_out, k_out=k_out)
    side.synchronize()
    check_16(q_out, *turned(*normed(q, w, EPS), positions, cos_sin, False))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm_rotate_qk(q, k, w, w, EPS, positions, cos_sin, q_out=q_out, k_out=k_out)
    for _ in range(4):
        q.copy_(heads(g, 5, 8, 128, dtype=BF16))
        positions.copy_(torch.randint(0, 100, (5,), generator=g))
        other = torch.randn(64, 64, device=dev) @ torch.randn(64, 64, device=dev)
        graph.replay()
        torch.cuda.synchronize()
        want = norm_rotate_qk(q, k, w, w, EPS, positions, cos_sin)
        assert torch.equal(q_out, want[0]) and torch.equal(k_out, want[1])
        del other


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("axes", [1, 3])
@pytest.mark.parametrize("dim", [128, 72, 90])
def test_a_token_alone_and_among_others(dev, dim, axes, dtype):
    """The same bits whatever else is in the batch."""
    g = torch.Generator().manual_seed(13)
    q, k = heads(g, 1100, 61, dim, dtype=dtype).to(dev), heads(g, 1100, 7, dim, dtype=dtype).to(dev)
    w = (torch.rand(dim, generator=g) + 0.5).to(dev)
    cos_sin = table(300, dim).to(dev)
    third = dim // 6
    turn = dict(sections=[dim // 2 - 2 * third, third, third], alternating=True) if axes == 3 else {}
    positions = torch.randint(0, 300, (axes, 1100) if axes == 3 else (1100,), generator=g).to(dev)
    for norm in (False, True):
        call = (lambda q, k, p: norm_rotate_qk(q, k, w, w, EPS, p, cos_sin, **turn)) if norm else (lambda q, k, p: rotate_qk(q, k, p, cos_sin, **turn))
        whole = call(q, k, positions)
        for at in (0, 517, 1099):
            one = call(q[at:at + 1], k[at:at + 1], positions[..., at:at + 1])
            assert torch.equal(one[0], whole[0][at:at + 1]) and torch.equal(one[1], whole[1][at:at + 1])


def test_gradients_and_tracers_are_refused(dev):
    from torch._subclasses.fake_tensor import FakeTensorMode

    cos_sin, positions = table(10, 64).to(dev), torch.arange(3, device=dev)
    x = torch.ones(3, 2, 64, device=dev, dtype=BF16)
    leaf = torch.ones(3, 2, 64, device=dev, dtype=BF16, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    for call in (lambda: rotate_qk(leaf, x, positions, cos_sin), lambda: rotate_qk(x, leaf, positions, cos_sin),
                 lambda: norm_rotate_qk(x, x, w, w, EPS, positions, cos_sin)):
        with pytest.raises(NotImplementedError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    with pytest.raises(NotImplementedError):
        torch.vmap(lambda q: rotate_qk(q, None, positions, cos_sin)[0])(torch.ones(4, 3, 2, 64, device=dev, dtype=BF16))
    with FakeTensorMode() as mode:
        with pytest.raises(NotImplementedError):
            rotate_qk(mode.from_tensor(x), None, mode.from_tensor(positions), mode.from_tensor(cos_sin))
    out = torch.empty_like(x)
    version = out._version
    rotate_qk(x, None, positions, cos_sin, q_out=out)
    assert out._version == version + 1
