"""A paged key / value cache in E4M3 or in 4 bits, and the operators that fill and read it.

``KVCache`` keeps E4M3 codes [pages, kv_heads, page, head_dim] and one
power-of-two float32 scale per block (page, head), for the keys and for the
values.  ``KVCache4`` keeps E2M1 codes, two a byte, and one E4M3 scale per 16
columns of a token: 9/16 of a byte a value.  The operators take either.  Which
page holds which tokens is the caller's plan:

  block_table  int32 [B, width]  the cache page of each page of a sequence
  lengths      int32 [B]         tokens the cache holds before the step
  counts       int32 [B]         new tokens of the step (None: all T)

``rope_append`` turns the query and key heads by their positions (lengths[b] +
t) and writes the new keys and values; ``attend`` then takes the same plan.
The plan stays on the device and is not read by the host: one that does not
fit (a count outside 0..T, tokens past the block table, a page outside the
cache) leaves the tokens concerned out and is reported by
``voyager_b200.check_errors()``.  There is no derivative: a backward pass that
reaches an output raises.

  rotary_table  cos / sin of every position, with the scalings for long contexts
  rope_append   (norms of the query and key heads +) rotary positions + append
  attend        causal attention of the newest tokens over the cache
  unpack        the codes of a 4-bit cache, one a byte
"""

import math
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from voyager_b200._launch import native

E4M3 = torch.float8_e4m3fn
PAGES = (32, 64, 128)
HEAD_DIMS = (64, 128)


@dataclass
class KVCache:
    """Codes float8_e4m3fn [pages, kv_heads, page, head_dim], scales float32
    [pages, kv_heads]."""

    k_codes: torch.Tensor
    v_codes: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, page: int = 64, device="cuda") -> "KVCache":
        """A cache that holds no token."""
        if page not in PAGES or head_dim not in HEAD_DIMS:
            raise ValueError(f"KVCache: page in {PAGES} and head_dim in {HEAD_DIMS}, not {page} and {head_dim}")
        c = [torch.zeros((pages, kv_heads, page, head_dim), dtype=torch.uint8, device=device).view(E4M3)
             for _ in range(2)]
        s = [torch.ones((pages, kv_heads), dtype=torch.float32, device=device) for _ in range(2)]
        return cls(c[0], c[1], s[0], s[1])


@dataclass
class KVCache4:
    """Codes uint8 [pages, kv_heads, page, head_dim / 2], two E2M1 codes a byte with
    the even column in the low half, scales float8_e4m3fn [pages, kv_heads, page,
    head_dim / 16], factors float32 [kv_heads] within 2^-100 .. 2^100.  A value is code x scale
    x its head's factor.  A block's scale is max|x| / (6 factor) as E4M3, with 4 significant
    bits from 2^-6 to 448; below, it loses bits down to its least, 2^-9.  So blocks
    up to 2688 x factor fit, those below 0.094 x factor are held more and more coarsely
    (scales up to a tenth off near 0.05 x factor, a third near 0.02), and below 0.012 x factor their codes
    shrink too.  A factor of max|x| / 2688 over a head uses the scales' whole range."""

    k_codes: torch.Tensor
    v_codes: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    k_factor: torch.Tensor
    v_factor: torch.Tensor

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, page: int = 64, device="cuda",
              k_factor: Optional[torch.Tensor] = None, v_factor: Optional[torch.Tensor] = None) -> "KVCache4":
        """A cache that holds no token; a factor of None is 1 for every head."""
        if page not in PAGES or head_dim not in HEAD_DIMS:
            raise ValueError(f"KVCache4: page in {PAGES} and head_dim in {HEAD_DIMS}, not {page} and {head_dim}")
        c = [torch.zeros((pages, kv_heads, page, head_dim // 2), dtype=torch.uint8, device=device) for _ in range(2)]
        s = [torch.ones((pages, kv_heads, page, head_dim // 16), device=device).to(E4M3) for _ in range(2)]
        f = [torch.ones(kv_heads, device=device) if f is None else f for f in (k_factor, v_factor)]
        return cls(*c, *s, *f)


Cache = Union[KVCache, KVCache4]


def _factors(cache: Cache):
    return (cache.k_factor, cache.v_factor) if isinstance(cache, KVCache4) else (None, None)


def rotary_table(positions: int, rotary_dim: int, theta: float = 10000.0, *, scaling: Optional[str] = None,
                 factor: float = 1.0, original: Optional[int] = None, low: float = 1.0, high: float = 32.0,
                 device="cuda") -> torch.Tensor:
    """float32 [positions, rotary_dim / 2, 2]: cos and sin of position x
    frequency, computed in float64.  Pair i has the frequency
    ``f_i = theta^(-2 i / rotary_dim)``.  ``scaling`` for contexts ``factor``
    times longer than the ``original`` one:

      None       positions as they are
      "linear"   positions divided by ``factor``
      "ntk"      theta times factor^(rotary_dim / (rotary_dim - 2)): the fastest
                 pair stays, the slowest turns ``factor`` times slower
      "parts"    by the turns n = original * f_i / (2 pi) that a pair makes in the
                 original context: pairs of ``high`` turns or more stay, of ``low``
                 or fewer are divided by ``factor``, between them a linear ramp in i
      "smooth"   the same with a ramp that is linear in n itself

    "parts" also multiplies cos and sin by 0.1 ln(factor) + 1, so that attention
    over longer contexts stays as sharp."""
    if rotary_dim < 2 or rotary_dim % 2 or positions < 0:
        raise ValueError(f"rotary_table: rotary_dim = {rotary_dim} must be even and positive, positions >= 0")
    if scaling not in (None, "linear", "ntk", "parts", "smooth"):
        raise ValueError(f"rotary_table: unknown scaling {scaling!r}")
    if factor < 1.0 or (scaling in ("parts", "smooth") and (not original or not 0 < low < high)):
        raise ValueError("rotary_table: factor >= 1; parts and smooth need the original context and 0 < low < high")
    f64 = dict(dtype=torch.float64, device=device)
    i = torch.arange(0, rotary_dim, 2, **f64)
    amp = 1.0
    if scaling == "ntk" and rotary_dim > 2:
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    freq = theta ** (-i / rotary_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "parts":
        # n(i) = original theta^(-i / rotary_dim) / 2 pi falls with i: the ramp's ends as indices
        at = [rotary_dim * math.log(original / (n * 2 * math.pi)) / (2 * math.log(theta)) for n in (high, low)]
        a = max(math.floor(at[0]), 0)
        b = min(math.ceil(at[1]), rotary_dim - 1)
        ramp = ((i / 2 - a) / max(b - a, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        amp = 0.1 * math.log(factor) + 1.0
    elif scaling == "smooth":
        n = original * freq / (2 * math.pi)
        keep = ((n - low) / (high - low)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
    angle = torch.arange(positions, **f64)[:, None] * freq
    return (torch.stack([angle.cos(), angle.sin()], -1) * amp).float()


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, cache: Cache,
                block_table: torch.Tensor, lengths: torch.Tensor, counts: Optional[torch.Tensor] = None,
                interleaved: bool = False, *, q_norm: Optional[torch.Tensor] = None,
                k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
    """Turn q [B, T, H, D] and k [B, T, Hkv, D] by ``table`` (``rotary_table``,
    at least block_table.shape[1] * page positions) at the positions
    lengths[b] + t, append k and v [B, T, Hkv, D] to the cache (in place), and
    return the turned q (0 for tokens past counts).  bfloat16 or float32;
    views such as the parts of one fused projection are read as they are.

    ``interleaved``: pairs are columns (2i, 2i + 1), otherwise (i, i +
    rotary_dim / 2); columns past rotary_dim stay.  ``q_norm`` / ``k_norm`` [D] in
    q's type: the heads of q / k are normalised first, ``x * rsqrt(mean(x^2) +
    eps) * weight`` over D in float32, unrounded before they turn.

    E4M3: a block's scale is the least power of two under which its tokens fit;
    it grows when a new token needs it, and the codes it holds are brought to the
    new scale.  4 bits: per 16 columns of a token ``scale = E4M3(max|x| / (6
    factor))``, at least 2^-9, and ``code = E2M1(x / (scale factor))``, to nearest
    even and saturating; what the cache holds is not touched."""
    return native.rope_append(q, k, v, table, cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale,
                              block_table, lengths, counts, interleaved, *_factors(cache), q_norm, k_norm, eps)


def attend(q: torch.Tensor, cache: Cache, block_table: torch.Tensor, lengths: torch.Tensor,
           counts: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention of the step's tokens over the cache, which holds their
    keys and values already (``rope_append`` with the same plan): q bfloat16
    [B, T, H, D] -> [B, T, H, D], row (b, t) over the keys 0 .. lengths[b] + t.
    ``scale`` defaults to 1 / sqrt(D).  Tokens past counts get 0."""
    return native.attend(q, cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale, block_table, lengths,
                         counts, scale, *_factors(cache))


def unpack(cache: KVCache4) -> Tuple[torch.Tensor, torch.Tensor]:
    """The key and value codes of a 4-bit cache as float8_e4m3fn [pages,
    kv_heads, page, head_dim], which holds every E2M1 value; scales and factors
    are not in them."""
    return native.unpack(cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale, *_factors(cache))
