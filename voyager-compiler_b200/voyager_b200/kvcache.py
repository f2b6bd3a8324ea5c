"""A paged key / value cache in E4M3, and the operators that fill and read it.

The cache keeps E4M3 codes [pages, kv_heads, page, head_dim] and one
power-of-two float32 scale per block (page, head), for the keys and for the
values.  Which page holds which tokens is the caller's plan:

  block_table  int32 [B, width]  the cache page of each page of a sequence
  lengths      int32 [B]         tokens the cache holds before the step
  counts       int32 [B]         new tokens of the step (None: all T)

``rope_append`` turns the query and key heads by their positions (lengths[b] +
t) and writes the new keys and values; ``attend`` then takes the same plan.
The plan stays on the device and is not read by the host: one that does not
fit (a count outside 0..T, tokens past the block table, a page outside the
cache) leaves the tokens concerned out and is reported by
``voyager_b200.check_errors()``.

  rotary_table  cos / sin of every position, with the scalings for long contexts
  rope_append   rotary positions + append
  attend        causal attention of the newest tokens over the cache
"""

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Optional

import torch

from voyager_b200 import _lib
from voyager_b200._launch import call, raw_stream

E4M3 = torch.float8_e4m3fn
PAGES = (32, 64, 128)
HEAD_DIMS = (64, 128)
_DTYPES = {torch.bfloat16: _lib.VQ_BF16, torch.float32: _lib.VQ_F32}
_I64x3, _I64x9 = ctypes.c_int64 * 3, ctypes.c_int64 * 9


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

    def check(self, what: str):
        """(pages, kv_heads, page, head_dim, device index); raises unless the
        four tensors are one cache on a CUDA device."""
        k, v, ks, vs = self.k_codes, self.v_codes, self.k_scale, self.v_scale
        if k.dtype != E4M3 or v.dtype != E4M3 or ks.dtype != torch.float32 or vs.dtype != torch.float32:
            raise NotImplementedError(f"{what}: a cache is float8_e4m3fn codes and float32 scales")
        shape = k.shape
        if len(shape) != 4 or v.shape != shape or ks.shape != shape[:2] or vs.shape != shape[:2]:
            raise ValueError(f"{what}: cache codes {tuple(shape)}, {tuple(v.shape)} and scales "
                             f"{tuple(ks.shape)}, {tuple(vs.shape)} are not one cache")
        pages, heads, page, dim = shape
        if page not in PAGES or dim not in HEAD_DIMS:
            raise NotImplementedError(f"{what}: page in {PAGES} and head_dim in {HEAD_DIMS}, not {page} and {dim}")
        if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
            raise ValueError(f"{what}: the cache's tensors must be contiguous")
        index = k.get_device()
        if v.get_device() != index or ks.get_device() != index or vs.get_device() != index:
            raise ValueError(f"{what}: the cache's tensors are on different devices")
        return pages, heads, page, dim, index


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


def _plan(what, index, B, block_table, lengths, counts):
    """(block_table's width, its pointer, lengths' and counts' pointers) after
    checks of the tensors; the values stay on the device."""
    for n, t, dim in (("block_table", block_table, 2), ("lengths", lengths, 1), ("counts", counts, 1)):
        if t is not None and (t.dtype != torch.int32 or t.dim() != dim or t.shape[0] != B
                              or t.get_device() != index or not t.is_contiguous()):
            raise ValueError(f"{what}: {n} must be contiguous int32 with {dim} dimension(s), the first {B}, "
                             f"on device {index}")
    return (block_table.shape[1], block_table.data_ptr(), lengths.data_ptr(),
            counts.data_ptr() if counts is not None else None)


def _heads(t, eb):
    """t [B, T, H, D] with a dense last dim and 16-byte rows, itself or a copy,
    and its strides."""
    b, h, s, d = t.stride()
    if d == 1 and not (t.data_ptr() | b * eb | h * eb | s * eb) & 15:
        return t, b, h, s
    t = t.clone(memory_format=torch.contiguous_format)
    return (t,) + t.stride()[:3]


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, cache: KVCache,
                block_table: torch.Tensor, lengths: torch.Tensor, counts: Optional[torch.Tensor] = None,
                interleaved: bool = False) -> torch.Tensor:
    """Turn q [B, T, H, D] and k [B, T, Hkv, D] by ``table`` (``rotary_table``,
    at least block_table.shape[1] * page positions) at the positions
    lengths[b] + t, append k and v [B, T, Hkv, D] to the cache (in place), and
    return the turned q (0 for tokens past counts).  bfloat16 or float32;
    views such as the parts of one fused projection are read as they are.

    ``interleaved``: pairs are columns (2i, 2i + 1), otherwise (i, i +
    rotary_dim / 2); columns past rotary_dim stay.  A block's scale is the
    least power of two under which its tokens fit E4M3; it grows when a new
    token needs it, and the codes it holds are brought to the new scale."""
    what = "rope_append"
    dtype = q.dtype
    code = _DTYPES.get(dtype)
    if code is None or k.dtype != dtype or v.dtype != dtype:
        raise NotImplementedError(f"{what}: q, k and v of one type, bfloat16 or float32")
    if not q.is_cuda:
        raise NotImplementedError(f"{what}: the CUDA kernel needs CUDA tensors")
    pages, Hkv, page, D, index = cache.check(what)
    shape = q.shape
    if len(shape) != 4 or shape[3] != D or k.shape != (shape[0], shape[1], Hkv, D) or v.shape != k.shape:
        raise ValueError(f"{what}: q {tuple(shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not match a "
                         f"cache of {Hkv} heads of {D}")
    B, T, H, _ = shape
    if H == 0 or H % Hkv:
        raise ValueError(f"{what}: {H} query heads do not group over {Hkv} kv heads")
    ts = table.shape
    if table.dtype != torch.float32 or len(ts) != 3 or ts[2] != 2 or not table.is_contiguous():
        raise ValueError(f"{what}: table must be contiguous float32 [positions, rotary_dim / 2, 2]")
    rot = 2 * ts[1]
    if rot == 0 or rot % 16 or rot > D:
        raise ValueError(f"{what}: rotary_dim = {rot} must be a multiple of 16 up to {D}")
    if (q.get_device() != index or table.get_device() != index or k.get_device() != index
            or v.get_device() != index):
        raise ValueError(f"{what}: operands on different devices")
    width, bt, held, new = _plan(what, index, B, block_table, lengths, counts)
    if ts[0] < width * page:
        raise ValueError(f"{what}: the table's {ts[0]} positions do not cover the block table's "
                         f"{width * page} tokens")
    eb = 2 if code == _lib.VQ_BF16 else 4
    q, qb, qt, qh = _heads(q, eb)
    k, kb, kt, kh = _heads(k, eb)
    v, vb, vt, vh = _heads(v, eb)
    out = q.new_empty(shape)
    call(_lib.load().vq_rope_append_kv8, index, what, q.data_ptr(), k.data_ptr(), v.data_ptr(),
         _I64x9(qb, qt, qh, kb, kt, kh, vb, vt, vh), code, table.data_ptr(), ts[0], rot, interleaved, B, T, H,
         Hkv, D, bt, width, held, new, pages, page, out.data_ptr(), cache.k_codes.data_ptr(),
         cache.v_codes.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr())
    return out


@functools.lru_cache(maxsize=512)
def _workspace_sizes(device: int, B, T, H, Hkv, D, page, width):
    f, c = ctypes.c_int64(), ctypes.c_int64()
    with torch.cuda.device(device):
        _lib.check(_lib.load().vq_attn_kv8_workspace(B, T, H, Hkv, D, page, width, ctypes.byref(f),
                                                     ctypes.byref(c)), "attend")
    return f.value, c.value


_counters = {}


def _join_counters(q, index, n):
    """Zeroed counters for a call on the current stream; each call leaves them
    zero, and calls on one stream do not overlap, so they share them.  A
    captured call gets its own, which live and die with its graph."""
    if torch.cuda.is_current_stream_capturing():
        return q.new_zeros(n, dtype=torch.int32)
    key = (index, raw_stream(index))
    t = _counters.get(key)
    if t is None or t.numel() < n:
        t = _counters[key] = q.new_zeros(max(n, 1024), dtype=torch.int32)
    return t


def attend(q: torch.Tensor, cache: KVCache, block_table: torch.Tensor, lengths: torch.Tensor,
           counts: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention of the step's tokens over the cache, which holds their
    keys and values already (``rope_append`` with the same plan): q bfloat16
    [B, T, H, D] -> [B, T, H, D], row (b, t) over the keys 0 .. lengths[b] + t.
    ``scale`` defaults to 1 / sqrt(D).  Tokens past counts get 0."""
    what = "attend"
    if q.dtype != torch.bfloat16:
        raise NotImplementedError(f"{what}: q must be bfloat16, not {q.dtype}")
    if not q.is_cuda:
        raise NotImplementedError(f"{what}: the CUDA kernel needs CUDA tensors")
    pages, Hkv, page, D, index = cache.check(what)
    shape = q.shape
    if len(shape) != 4 or shape[3] != D or shape[2] == 0 or shape[2] % Hkv:
        raise ValueError(f"{what}: q {tuple(shape)} does not match a cache of {Hkv} heads of {D}")
    if q.get_device() != index:
        raise ValueError(f"{what}: operands on different devices")
    B, T, H, _ = shape
    width, bt, held, new = _plan(what, index, B, block_table, lengths, counts)
    q, qb, qt, qh = _heads(q, 2)
    out = q.new_empty(shape)
    floats, n = _workspace_sizes(index, B, T, H, Hkv, D, page, width)
    done = _join_counters(q, index, n)
    part = q.new_empty(floats, dtype=torch.float32)
    call(_lib.load().vq_attn_kv8, index, what, q.data_ptr(), _I64x3(qb, qt, qh), B, T, H, Hkv, D,
         cache.k_codes.data_ptr(), cache.v_codes.data_ptr(), cache.k_scale.data_ptr(),
         cache.v_scale.data_ptr(), pages, page, bt, width, held, new,
         1.0 / math.sqrt(D) if scale is None else scale, part.data_ptr(), floats,
         done.data_ptr(), done.numel(), out.data_ptr())
    return out
