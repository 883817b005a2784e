"""The row-scaled operators restated in 64 bits, with how far 32-bit arithmetic may take their results (row_out.h, moe_few.hip and
the GEMM epilogues have the arithmetic that the bounds count)."""
import torch

U = 2.0 ** -24  # half a step of float32, relative
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}  # half of the smallest half (bfloat16 has float32's exponents)


def rms(x, w, eps, res=None):
    v = x.double() if res is None else x.double() + res.double()
    return v, v / torch.sqrt((v * v).mean(dim=-1, keepdim=True) + eps) * w.double()


def rms_error(n):
    """Relative error of y: a sum of n squares over at least 64 lanes (n / 64 additions in a lane, six between lanes and one
    between waves; at most 256 lanes' share where 1024 work), halved by the root; six further operations."""
    return (0.5 * (n / 64 + 12) + 8) * U


def silu_mul(x):
    gate, up = x.double().chunk(2, dim=-1)
    return gate * torch.sigmoid(gate) * up


def silu_error(x):
    """Relative error of an element of y: exp2's argument (|gate| * 1.45 roundings of 2^-24, times ln 2) and its last place, the
    sum, the reciprocal (a step each) and two products."""
    gate = x.double().chunk(2, dim=-1)[0].abs()
    return (1.5 * gate + 10) * 2 * U


def symmetric(y, int8):
    amax = y.abs().amax(dim=-1, keepdim=True)
    return amax.clamp_min(1e-10) / 127 if int8 else amax / 448


def asymmetric(y):
    lo, hi = y.amin(dim=-1, keepdim=True).clamp_max(0), y.amax(dim=-1, keepdim=True).clamp_min(0)
    scale = (hi - lo).clamp_min(1e-10) / 255
    return scale, -128 - lo / scale


def check_codes(y, error, q, s, zp=None, fixed=None):
    """Codes, scales and zero points of rows whose 64-bit values are y, known in 32 bits to `error` (relative, broadcastable)."""
    error = error + 8 * U  # the scale's division, the multiplier's, the product and its clamp
    worst = error.amax(dim=-1, keepdim=True) if torch.is_tensor(error) else error
    assert s.dtype == torch.float32 and s.shape == (y.shape[0], 1)
    s64 = s.double().cpu()
    if fixed is not None:
        assert torch.equal(s.cpu(), torch.full_like(s.cpu(), fixed))
    elif zp is None:
        want = symmetric(y, q.dtype == torch.int8)
        assert ((s64 - want).abs() <= want * worst).all(), ((s64 - want).abs() / want).max()
    else:
        want, z64 = asymmetric(y)
        assert ((s64 - want).abs() <= want * worst).all()
        z = zp.cpu()
        assert zp.dtype == torch.int32 and zp.shape == s.shape
        assert ((z - z64).abs() <= 0.5 + 255 * worst).all() and z.min() >= -128 and z.max() <= 127
    if q.dtype == torch.int8:
        back = s64 * (q.cpu().double() - (0 if zp is None else zp.cpu().double()))
        off = (back - y).abs() - y.abs() * error
        assert (off <= s64 * (0.5 + 255 * 4 * U)).all(), (off / s64).max()
        if zp is not None:
            zero = y == 0
            assert (q.cpu()[zero] == zp.cpu().expand_as(q)[zero]).all()  # zeros are kept
    else:
        code = q.cpu().float().double()
        clamped = (y / torch.where(s64 == 0, torch.ones_like(s64), s64)).clamp(-448, 448)
        # half a step of e4m3: 2^-4 relative, 2^-10 among its smallest numbers
        slack = clamped.abs() * error
        bound = torch.maximum((clamped.abs() + slack) * 2.0 ** -4, torch.full_like(clamped, 2.0 ** -10)) + slack
        assert ((code - clamped).abs() <= bound).all(), ((code - clamped).abs() / bound).max()


def check_rounded(out, want, error, extra=0.0):
    """A 16-bit result of a 64-bit value known to `error` (relative) and `extra` (absolute)."""
    t = out.dtype
    off = (out.double().cpu() - want).abs()
    bound = want.abs() * (error + HALF_STEP[t] * (1 + error)) + extra * (1 + HALF_STEP[t]) + LEAST[t]
    assert (off <= bound).all(), (off / bound.clamp_min(1e-300)).max()


def check_product(out, codes, zp, w, sa, sb, bias):
    """out [M, N] of int8 codes [M, K], zero points [M, 1] or None, weight rows [N, K]: the sum is exact, its conversion, the
    product of the scales, theirs and the bias's addition round."""
    c = codes.double() - (0 if zp is None else zp.double())
    acc = torch.matmul(c, w.double().t())
    scale = sa.double().view(-1, 1) * sb.double().view(1, -1)
    want = acc * scale
    extra = want.abs() * 4 * U
    if bias is not None:
        extra = (want.abs() * 4 + bias.double().abs()) * U
        want = want + bias.double()
    check_rounded(out, want.cpu(), U, extra.cpu())


def experts(x, xs, w1, w2, s1, s2, weights, ids, b1=None, b2=None, factor=1.0):
    """(out [M, H] in 64 bits, how far 32-bit arithmetic may be from it).  Codes of an intermediate value within its own error
    of the border between two steps may fall on either side; their step, times their weights, is what that costs."""
    m, h = x.shape
    e_count, two_i = w1.shape[:2]
    half = two_i // 2
    out, off = torch.zeros(m, h, dtype=torch.float64), torch.zeros(m, h, dtype=torch.float64)
    int8 = x.dtype == torch.int8
    xd = x.double() if int8 else x.float().double()
    for t in range(m):
        for k in range(ids.shape[1]):
            e = int(ids[t, k])
            if not 0 <= e < e_count:
                continue
            wd = w1[e].double() if int8 else w1[e].float().double()
            scale = xs.double().view(-1)[t] * s1[e].double().view(-1)
            terms = wd.abs() @ xd[t].abs()
            acc = wd @ xd[t]
            # a lane adds an eighth of the row, two at a time in the e4m3 form, then three to five sums between lanes (int8: exact)
            err = (0.0 if int8 else (h / 8 + 8)) * U * terms * scale
            hv = acc * scale
            if b1 is not None:
                hv = hv + b1[e].double()
                err = err + hv.abs() * U
            err = err + (acc * scale).abs() * 4 * U
            g, u = hv[:half], hv[half:]
            a = g * torch.sigmoid(g) * u
            # |d silu / d g| is below 1.1; expf, a sum, a division and a product on top
            ea = u.abs() * 1.1 * err[:half] + (g * torch.sigmoid(g)).abs() * err[half:] + err[:half] * err[half:] * 1.1 + a.abs() * 8 * U
            s = symmetric(a.view(1, -1), int8)[0, 0]
            if s == 0:  # a row of zeros, in e4m3
                if b2 is not None:
                    out[t] += b2[e].double() * weights[t, k].double()
                continue
            es = ea.max() / (127 if int8 else 448) + s * 4 * U
            v = a / s
            ev = ea / s + v.abs() * (es / s) + v.abs() * 8 * U
            if int8:
                code = torch.sign(v) * torch.floor(v.abs() + 0.5)
                step = torch.ones_like(v)
                border = (v.abs() + 0.5) - torch.floor(v.abs() + 0.5)
                near = torch.minimum(border, 1 - border) <= ev
            else:
                step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))).clamp(-6, 8) - 3)
                code = torch.round(v / step) * step
                near = ((v / step - torch.floor(v / step)) - 0.5).abs() * step <= ev
            w2d = w2[e].double() if int8 else w2[e].float().double()
            s2d = s2[e].double().view(-1)
            row = (w2d @ code) * s * s2d
            eo = (w2d.abs() @ (step * near)) * s * s2d + row.abs() * (es / s + 5 * U)
            eo = eo + (0.0 if int8 else (half / 8 + 8)) * U * (w2d.abs() @ code.abs()) * s * s2d
            if b2 is not None:
                row = row + b2[e].double()
                eo = eo + row.abs() * U
            wt = weights[t, k].double()
            out[t] += row * wt
            off[t] += (eo + row.abs() * (ids.shape[1] + 2) * U) * wt.abs()
    return out * factor, (off + out.abs() * 2 * U) * abs(factor)
