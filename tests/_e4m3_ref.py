"""64-bit references of the cached-decoding operators (test infrastructure)."""

import math

import torch

E4M3 = torch.float8_e4m3fn


def e4m3(x):
    """float64 -> the nearest E4M3 value, ties to even, saturating."""
    e = torch.frexp(x.abs().clamp(min=1e-300))[1].double() - 1
    step = torch.exp2(e.clamp(min=-6) - 3)
    return torch.where(x.isnan(), x, ((x / step).round() * step).clamp(-448, 448))


def check_codes(codes, q, delta):
    """Each code is the rounding of some value within `delta` (relative) of the exact quotient q."""
    c = codes.double()
    assert torch.equal(c.isnan(), q.isnan())
    ok = q.isnan() | ((c >= torch.minimum(e4m3(q * (1 - delta)), e4m3(q * (1 + delta))))
                      & (c <= torch.maximum(e4m3(q * (1 - delta)), e4m3(q * (1 + delta)))))
    assert bool(ok.all()), (c[~ok][:4], q[~ok][:4])


def check_close(got, want, bound):
    """|got - want| <= bound, elementwise; NaN in the same places."""
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan())
    bad = ~want.isnan() & ~((got - want).abs() <= bound)
    assert not bool(bad.any()), (int(bad.sum()), got[bad][:4], want[bad][:4], bound.expand_as(want)[bad][:4])


def check_rounded(got, want, err):
    """got (of its type) lies between the roundings of want - err and want + err."""
    lo, hi = ((want + e).to(got.dtype).double() for e in (-err, err))
    g = got.double()
    ok = (g >= lo) & (g <= hi) | want.isnan() & g.isnan()
    assert bool(ok.all()), (int((~ok).sum()), g[~ok][:4], want[~ok][:4])


def pow2_scale(amax):
    """The least power of two with amax / s <= 448, in [2^-100, 2^120] (python floats)."""
    if amax == 0:
        return 2.0 ** -100
    if amax == math.inf:
        return 2.0 ** 120
    m, e = math.frexp(amax)
    return 2.0 ** min(max(e - 9 + (m > 0.875), -100), 120)


def rotate(x, table, pos, interleaved):
    """x [T, heads, D] float64 turned at positions pos [T]."""
    rot = 2 * table.shape[1]
    cs = table.double()[pos][:, None]
    h = torch.arange(rot // 2, device=x.device)
    a, b = (2 * h, 2 * h + 1) if interleaved else (h, h + rot // 2)
    z = torch.complex(x[..., a], x[..., b]) * torch.complex(cs[..., 0], cs[..., 1])
    x = x.clone()
    x[..., a], x[..., b] = z.real, z.imag
    return x


def attention(q, k, v, held, scale):
    """q [T, G, D], k and v [keys, D] float64: the output and sum_j p_j |v_j|."""
    T, G, D = q.shape
    s = torch.einsum("tgd,kd->tgk", q, k) * scale
    late = torch.arange(k.shape[0], device=q.device) > held + torch.arange(T, device=q.device)[:, None]
    p = torch.softmax(s.masked_fill(late[:, None], -math.inf), -1)
    out = torch.empty_like(q)
    for t in range(T):  # a value that a row does not see does not enter, be it NaN
        n = held + t + 1
        out[t] = p[t, :, :n] @ v[:n]
    return out, p @ torch.nan_to_num(v).abs()
