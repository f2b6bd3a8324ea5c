"""64-bit references of the 4-bit cache's operators (test infrastructure)."""

import torch

from _e4m3_ref import e4m3

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK = 16


def e2m1(x):
    """float64 -> the nearest E2M1 value, ties to the even code, saturating."""
    a = x.abs().clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0)).double()
    return torch.where(x.isnan(), x, torch.copysign((a / step).round() * step, x))


def block_scale(amax, factor):
    """E4M3(amax / (6 factor)), at least 2^-9."""
    s = e4m3(amax / (6.0 * factor))
    return torch.where(s.isnan(), s, s.clamp(min=2.0 ** -9))


def codes_of(raw):
    """Packed uint8 [.., n] -> float64 values [.., 2 n]."""
    lut = torch.tensor(E2M1 + tuple(-x for x in E2M1), dtype=torch.float64, device=raw.device)
    return torch.stack([lut[(raw & 15).long()], lut[(raw >> 4).long()]], -1).flatten(-2)


def values_of(raw, scale, factor):
    """Packed codes [.., D / 2], E4M3 scales [.., D / 16] and a factor that broadcasts to [.., 1] -> float64."""
    x = codes_of(raw).unflatten(-1, (-1, BLOCK))
    return (x * (scale.double() * factor)[..., None]).flatten(-2)


def head_norm(x, weight, eps):
    """x [.., D] float64 normalised over D; no weight: as it is."""
    if weight is None:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
