"""Edges of the cached-decoding operators: plans that do not fit, empty
caches, blocks whose scale grows, streams, gradients, values at the ends of
float32's range.

Tolerances.  Attention: softmax weights are held in f16 (2^-11 relative),
scores are float32 sums of f16 products (below 2^-13 of a weight at these
sizes), so an output is within 2^-10 of sum_j p_j |v_j|, and one bf16 rounding
(2^-8).  What is a power of two or a copy is compared for equality."""

import math

import pytest
import torch

from _e4m3_ref import E4M3, check_close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _setup():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    import voyager_b200  # noqa: F401

    yield


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cache(pages, Hkv, page, D, seed):
    from voyager_b200 import kvcache

    g = _gen(seed)
    c = kvcache.KVCache.empty(pages, Hkv, D, page)
    for t, s in ((c.k_codes, c.k_scale), (c.v_codes, c.v_scale)):
        t.copy_((torch.randn(t.shape, generator=g, device="cuda") * 100).clamp(-448, 448))
        s.copy_(torch.exp2(torch.randint(-9, -3, s.shape, generator=g, device="cuda").float()))
    return c


# ---------------------------------------------------------------------------
def _attention_without(q, cache, bt, b, h, held, n):
    """The n newest tokens' attention over head h in float64, the keys of pages
    outside the cache left out; and sum_j p_j |v_j|.  q [n, G, D]."""
    pages, _, page, D = cache.k_codes.shape
    end = held + n
    pos = torch.arange(end, device="cuda")
    pid = bt[b].long()[pos // page]
    there = (pid >= 0) & (pid < pages)
    pid = torch.where(there, pid, 0)
    k, v = (c[:, h].view(torch.uint8)[pid, pos % page].view(E4M3).double() * s[pid, h, None].double()
            for c, s in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)))
    k, v = (torch.where(there[:, None], x, 0.0) for x in (k, v))
    s = torch.einsum("tgd,kd->tgk", q, k) / math.sqrt(D)
    seen = there & (pos <= held + torch.arange(n, device="cuda")[:, None])
    s = s.masked_fill(~seen[:, None], -math.inf)
    p = torch.where(seen.any(-1)[:, None, None], torch.softmax(s, -1), 0.0)
    return p @ v, p @ v.abs()


@pytest.mark.parametrize("fill", ["codes", "nan"])
@pytest.mark.parametrize("D,page", [(128, 64), (64, 32), (128, 128)])
@pytest.mark.parametrize("T,G", [(1, 4), (5, 4), (3, 1), (1, 16)])
def test_attend_leaves_out_pages_outside_the_cache(T, G, D, page, fill):
    """The keys of such a page (first, middle, last, all of a sequence's) are
    left out whatever page 0 holds, and the call is reported."""
    import voyager_b200
    from voyager_b200 import _lib, kvcache

    width, Hkv = 9, 2
    held = [page * 9 - T, page * 7 + 3, page * 4, 2 * page - 1, page + 5]
    B = len(held)
    cache = _cache(B * width + 1, Hkv, page, D, T * G + D)
    pages = cache.k_codes.shape[0]
    bt = 1 + torch.randperm(B * width, generator=_gen(1), device="cuda").view(B, width).int()
    for c, s in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)):
        if fill == "nan":
            c.view(torch.uint8)[0] = 0x7F
            s[0] = math.nan
        else:
            c[0] = 448.0
            s[0] = 2.0
    bt[0, 0] = -1
    bt[0, 5] = pages
    bt[1, 7] = 1 << 30          # the newest tokens' page
    bt[2, 1:4] = -(1 << 31)
    bt[3, :] = -1
    q = torch.randn(B, T, Hkv * G, D, generator=_gen(2), device="cuda").bfloat16()
    out = kvcache.attend(q, cache, bt, _i32(held))
    with pytest.raises(_lib.VqError, match="plan"):
        voyager_b200.check_errors()
    for b in range(B):
        for h in range(Hkv):
            want, mag = _attention_without(q[b, :, h * G:(h + 1) * G].double(), cache, bt, b, h, held[b], T)
            check_close(out[b, :, h * G:(h + 1) * G], want, mag * 2.0 ** -10 + want.abs() * 2.0 ** -8)
    assert not bool(out[3].any())


def test_attend_leaves_out_pages_in_long_heads():
    """The same where a head is cut into pieces, one of them of such pages only."""
    import voyager_b200
    from voyager_b200 import _lib, kvcache

    page, D, G, held = 64, 128, 4, 30000
    width = held // page + 1
    cache = _cache(width + 1, 1, page, D, 5)
    cache.k_codes[0], cache.v_codes[0] = 448.0, 448.0
    bt = 1 + torch.randperm(width, generator=_gen(3), device="cuda").view(1, width).int()
    bt[0, 100:180] = -1
    bt[0, ::7] = width + 1
    q = torch.randn(1, 1, G, D, generator=_gen(4), device="cuda").bfloat16()
    out = kvcache.attend(q, cache, bt, _i32([held]))
    with pytest.raises(_lib.VqError, match="plan"):
        voyager_b200.check_errors()
    want, mag = _attention_without(q[0].double(), cache, bt, 0, 0, held, 1)
    check_close(out[0], want, mag * 2.0 ** -10 + want.abs() * 2.0 ** -8)
