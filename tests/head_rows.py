"""Heads between a projection and its attention restated in 64 bits, with how far 32-bit arithmetic may take their results
(head_rows.hip has the arithmetic that the bounds count)."""
import torch

from tests.row_layers import HALF_STEP, LEAST, U

F8 = torch.float8_e4m3fn


def pair_axes(half, sections, alternating):
    """The axis of each pair; with one axis all zeros."""
    if sections is None:
        return [0] * half
    if alternating:
        n = len(sections)
        return [i % n if i < n * sections[i % n] else 0 for i in range(half)]
    return [a for a, count in enumerate(sections) for _ in range(count)]


def turned(y, off, positions, cos_sin, interleaved, sections=None, alternating=False):
    """(rotated, off) of y [tokens, heads, dim], known to `off` (absolute), all in 64 bits on the CPU: two products and their sum
    round by 2^-24 of the products' magnitudes."""
    half = cos_sin.shape[1] // 2
    pos = positions.cpu().view(1, -1) if positions.dim() == 1 else positions.cpu()
    table = cos_sin.cpu().double()
    at = pos[torch.tensor(pair_axes(half, sections, alternating), dtype=torch.long)].t().long()  # [tokens, pairs]
    good = (at >= 0) & (at < table.shape[0])
    pair = torch.arange(half)
    safe = at.clamp(0, max(table.shape[0] - 1, 0))
    nan = torch.full_like(good, 0, dtype=torch.float64) + float("nan")
    c = torch.where(good, table[safe, pair], nan).unsqueeze(1)
    s = torch.where(good, table[safe, pair + half], nan).unsqueeze(1)
    out, err = y.clone(), off.clone()
    first = slice(0, half) if not interleaved else slice(0, 2 * half, 2)
    second = slice(half, 2 * half) if not interleaved else slice(1, 2 * half, 2)
    a, b, ea, eb = y[..., first], y[..., second], off[..., first], off[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    err[..., first] = (a * c).abs() * 2 * U + (b * s).abs() * 2 * U + ea * c.abs() + eb * s.abs()
    err[..., second] = (b * c).abs() * 2 * U + (a * s).abs() * 2 * U + eb * c.abs() + ea * s.abs()
    return out, err * (1 + 4 * U)


def normed(x, weight, eps):
    """(y, off): a lane adds 16 squares, six sums between lanes, the division and epsilon, halved by the root; the root's last
    place, two products."""
    v = x.cpu().double()
    if weight is None:
        return v, torch.zeros_like(v)
    y = v / torch.sqrt((v * v).mean(dim=-1, keepdim=True) + eps) * weight.cpu().double()
    return y, y.abs() * (0.5 * (16 + 6 + 3) + 2 + 2) * U


def check_16(out, want, off):
    t = out.dtype
    got = out.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    fine = ~torch.isnan(want)
    bound = (off + HALF_STEP[t] * (want.abs() + off) + LEAST[t])[fine]
    miss = (got - want).abs()[fine]
    assert (miss <= bound).all(), (miss / bound.clamp_min(1e-300)).max()


def check_8(codes, want, off, given=None, scales=None, group=None):
    """8-bit codes of rows whose 64-bit values are `want` [..., dim]: with a given scale (broadcastable to want), or with the scales
    that came back [..., dim / group]."""
    group = group or want.shape[-1]
    grouped = lambda t: t.reshape(*t.shape[:-1], t.shape[-1] // group, group)  # noqa: E731
    int8 = codes.dtype == torch.int8
    value = codes.cpu().double() if int8 else codes.cpu().float().double()
    if given is None:
        s = scales.cpu().double().unsqueeze(-1)
        amax = grouped(want).abs().amax(dim=-1, keepdim=True)
        exact = amax.clamp_min(1e-10) / 127 if int8 else amax / 448
        assert ((s - exact).abs() <= grouped(off).amax(dim=-1, keepdim=True) / (127 if int8 else 448) + exact * 2 * U).all()
        s = s.expand(grouped(want).shape).reshape(want.shape)
    else:
        s = given.cpu().double().expand(want.shape)
    v = want / torch.where(s == 0, torch.ones_like(s), s)
    slack = off / s.clamp_min(1e-300) + v.abs() * 4 * U
    if int8:
        assert ((value - v).abs() <= 0.5 + slack).all(), ((value - v).abs() - 0.5).max()
        return
    clamped = v.clamp(-448, 448)
    bound = torch.maximum((clamped.abs() + slack) * 2.0 ** -4, torch.full_like(v, 2.0 ** -10)) + slack
    assert ((value - clamped).abs() <= bound).all(), ((value - clamped).abs() / bound).max()


def table(rows, width, dtype=torch.float32, base=10000.0):
    angle = torch.arange(rows, dtype=torch.float64).view(-1, 1) * base ** (torch.arange(0, width, 2, dtype=torch.float64) / -width)
    return torch.cat([angle.cos(), angle.sin()], dim=-1).to(dtype)


def heads(g, *shape, dtype):
    return (torch.randn(*shape, generator=g) * torch.exp(0.7 * torch.randn(shape[-1], generator=g))).to(dtype)
