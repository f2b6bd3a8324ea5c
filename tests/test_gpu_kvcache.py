"""Rotary positions, the append to the E4M3 cache and attention over it,
against the formulas in 64 bits.

Tolerances.  Rotation: two float32 products and a sum, 3 * 2^-24 of |a| + |b|
: q must be the rounding of a value within that of the exact one, and a key's code
the E4M3 rounding of a value within it of the exact quotient.  Attention: weights are held in f16 (2^-11
relative), scores are float32 sums of f16 products (below 2^-13 of a weight at
these sizes), so an output is within 2^-10 of sum_j p_j |v_j|, and one bf16
rounding (2^-8)."""

import math

import pytest
import torch

from _e4m3_ref import E4M3, attention, check_close, check_rounded, e4m3, pow2_scale, rotate

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


def _cache(pages, Hkv, page, D, seed, stale=None):
    """Random codes and scales; `stale`: every byte that value instead."""
    from voyager_b200 import kvcache

    g = _gen(seed)
    c = kvcache.KVCache.empty(pages, Hkv, D, page)
    for t, s in ((c.k_codes, c.k_scale), (c.v_codes, c.v_scale)):
        if stale is None:
            t.copy_((torch.randn(t.shape, generator=g, device="cuda") * 100).clamp(-448, 448))
        else:
            t.view(torch.uint8).fill_(stale)
        s.copy_(torch.exp2(torch.randint(-9, -3, s.shape, generator=g, device="cuda").float()))
    return c


def _table(B, width, seed, extra=2):
    g = _gen(seed)
    return torch.randperm(B * width + extra, generator=g, device="cuda")[:B * width].reshape(B, width).int().contiguous()


# ---------------------------------------------------------------------------
def _check_append(B, T, Hkv, G, D, page, held, counts, rot, interleaved, dtype=torch.bfloat16, seed=0, values=None,
                  fused=True):
    from voyager_b200 import kvcache

    g = _gen(seed)
    H = Hkv * G
    width = max(1, -(-max(h + T for h in held) // page))
    qkv = torch.randn(B, T, H + 2 * Hkv, D, generator=g, device="cuda") * 2
    if values is not None:
        values(qkv)
    qkv = qkv.to(dtype)
    q, k, v = qkv.split([H, Hkv, Hkv], 2)
    if not fused:
        q, k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    table = kvcache.rotary_table(width * page, rot, scaling="linear", factor=2.0)
    bt = _table(B, width, seed + 1)
    cache = _cache(B * width + 2, Hkv, page, D, seed + 2)
    was = [t.clone() for t in (cache.k_codes.view(torch.uint8), cache.v_codes.view(torch.uint8), cache.k_scale,
                               cache.v_scale)]
    out = kvcache.rope_append(q, k, v, table, cache, bt, _i32(held), _i32(counts) if counts is not None else None,
                              interleaved)
    assert out.shape == q.shape and out.dtype == dtype
    touched = [torch.zeros_like(w, dtype=torch.bool) for w in was]
    for b in range(B):
        h, n = held[b], counts[b] if counts is not None else T
        assert not bool(out[b, n:].any())
        if n == 0:
            continue
        pos = torch.arange(h, h + n, device="cuda")
        wq = rotate(q[b, :n].double(), table, pos, interleaved)
        mag = q[b, :n].double().abs().amax(-1, keepdim=True) * 2
        check_rounded(out[b, :n], wq, mag * 3 * 2.0 ** -24)
        turned = rotate(k[b, :n].double(), table, pos, interleaved)
        # float32 throughout: what it cannot hold is an infinity, and saturates
        turned = torch.where(turned.abs() > torch.finfo(torch.float32).max, turned.sign() * math.inf, turned)
        vals = (turned, v[b, :n].double())
        for i, (codes, scale) in enumerate(((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale))):
            for p in range(h // page, (h + n - 1) // page + 1):
                lo, hi, old, pid = max(h, p * page), min(h + n, (p + 1) * page), max(0, h - p * page), int(bt[b, p])
                for hd in range(Hkv):
                    x = vals[i][lo - h:hi - h, hd]
                    top = float(torch.nan_to_num(x.abs(), 0.0, posinf=math.inf).max())
                    s0 = float(was[2 + i][pid, hd]) if old else 0.0
                    s = float(scale[pid, hd])
                    near = {max(pow2_scale(top * (1 + d)), s0) for d in (-1e-6, 0.0, 1e-6)}
                    assert s in near, (s, near)
                    c = codes[pid, hd].double()
                    err = 0.0
                    new = c[lo - p * page:hi - p * page]
                    quo = x / s
                    if i == 0:
                        err = float(k[b, :n, hd].double().abs().nan_to_num(0.0, posinf=0.0).amax()) * 6 * 2.0 ** -24 / s
                    nan = quo.isnan()
                    assert torch.equal(new.isnan(), nan)
                    ok = nan | ((new >= e4m3(quo - err)) & (new <= e4m3(quo + err)))
                    assert bool(ok.all()), (new[~ok][:4], quo[~ok][:4])
                    if old:
                        o = was[i].view(E4M3)[pid, hd, :old].double()
                        assert torch.equal(c[:old], e4m3(o * (s0 / s)))
                    touched[i][pid, hd, :hi - p * page] = True
                    touched[2 + i][pid, hd] = True
    for t, w, now in zip(touched, was, (cache.k_codes.view(torch.uint8), cache.v_codes.view(torch.uint8), cache.k_scale,
                                        cache.v_scale)):
        assert torch.equal(now[~t], w[~t])  # nothing else changed


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot,page", [(128, 128, 64), (128, 32, 128), (64, 64, 32), (64, 16, 64), (128, 96, 32),
                                        (64, 48, 128)])
def test_append_single_tokens(D, rot, page, interleaved):
    held = [0, 1, page - 1, page, 3 * page + 5]
    _check_append(5, 1, 2, 3, D, page, held, None, rot, interleaved, seed=D + rot)
    _check_append(5, 1, 2, 3, D, page, held, [1, 0, 1, 1, 0], rot, interleaved, torch.float32, seed=D + page)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,page,D", [(2, 32, 64), (31, 32, 128), (33, 32, 128), (64, 64, 64), (130, 64, 128),
                                      (257, 128, 128), (200, 128, 64)])
def test_append_prompts(T, page, D, dtype):
    """Prompts over several pages, from every kind of start, of unequal counts."""
    _check_append(4, T, 2, 1, D, page, [0, 7, page - 1, 2 * page], [T, T - 1, T, T // 2], D, False, dtype, seed=T)
    _check_append(2, T, 1, 2, D, page, [5, 0], None, D // 2, True, dtype, seed=T + 1, fused=False)


def test_append_scale_growth_and_specials():
    """Values far above the block's scale (its codes are brought to the new
    one), blocks of zeros, NaN, infinities and the range's ends."""
    def big(x):
        x[0] *= 300.0
        x[1] *= 1e-30
        x[2] = 0.0

    _check_append(4, 3, 2, 1, 128, 64, [9, 70, 3, 62], None, 128, False, seed=3, values=big)

    def special(x):
        x[0, 0, -1, 5] = float("nan")   # v
        x[1, 0, -1, 7] = float("inf")
        x[2, :, 1:] = 3e38
        x[3, :, 1:] = 1e-38

    _check_append(4, 2, 1, 1, 64, 32, [0, 4, 40, 64], None, 16, True, torch.float32, seed=4, values=special)


def test_append_token_by_token_is_the_prompt():
    """Appending one token at a time gives the prompt's blocks: the same scales,
    and codes equal but for those that turned subnormal on the way."""
    from voyager_b200 import kvcache

    g = _gen(5)
    T, Hkv, D, page = 150, 2, 128, 64
    x = torch.randn(1, T, 3 * Hkv, D, generator=g, device="cuda") * torch.linspace(0.01, 4, T, device="cuda")[:, None, None]
    q, k, v = x.bfloat16().split(Hkv, 2)
    table = kvcache.rotary_table(192, D)
    bt = _i32([[2, 0, 1]])
    whole, steps = (kvcache.KVCache.empty(3, Hkv, D, page) for _ in range(2))
    qw = kvcache.rope_append(q, k, v, table, whole, bt, _i32([0]))
    qs = [kvcache.rope_append(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], table, steps, bt, _i32([t])) for t in range(T)]
    assert torch.equal(torch.cat(qs, 1), qw)
    for n in ("k", "v"):
        s, s2 = getattr(whole, n + "_scale"), getattr(steps, n + "_scale")
        assert torch.equal(s, s2)
        a, b = getattr(whole, n + "_codes").double(), getattr(steps, n + "_codes").double()
        assert float((a - b).abs().max()) <= 2.0 ** -9  # one subnormal step
        assert torch.equal(a[a.abs() >= 2.0 ** -5], b[a.abs() >= 2.0 ** -5])


def test_plan_errors_are_reported():
    """Plans that do not fit leave the tokens out, touch nothing outside and
    set the sticky word."""
    import voyager_b200
    from voyager_b200 import _lib, kvcache

    def go(held, counts, bt):
        cache = _cache(4, 1, 32, 64, 6)
        before = cache.k_codes.view(torch.uint8).clone()
        q = torch.ones(1, 2, 1, 64, device="cuda").bfloat16()
        kvcache.rope_append(q, q, q, kvcache.rotary_table(64, 64), cache, bt, _i32([held]), _i32([counts]))
        with pytest.raises(_lib.VqError, match="plan"):
            voyager_b200.check_errors()
        a = kvcache.attend(q, cache, bt, _i32([held]), _i32([counts]))
        with pytest.raises(_lib.VqError, match="plan"):
            voyager_b200.check_errors()
        assert a.shape == q.shape
        return int((cache.k_codes.view(torch.uint8) != before).any(-1).sum())

    ok = _i32([[1, 2]])
    assert go(3, 3, ok) == 2      # clamped to the two tokens there are
    assert go(-1, 1, ok) == 0
    assert go(3, -2, ok) == 0
    assert go(63, 2, ok) == 1     # one slot left
    assert go(1000, 1, ok) == 0
    assert go(3, 1, _i32([[-1, 2]])) == 0
    assert go(3, 1, _i32([[4, 2]])) == 0
    voyager_b200.check_errors()


# ---------------------------------------------------------------------------
def _check_attend(B, T, Hkv, G, D, page, held, counts=None, seed=0, scale=None, stale=None, cache=None, bt=None,
                  sharp=1.0, edit=None, strided=False):
    from voyager_b200 import kvcache

    H = Hkv * G
    width = max(1, -(-max(h + T for h in held) // page))
    bt = _table(B, width, seed + 1) if bt is None else bt
    cache = _cache(int(bt.max()) + 2, Hkv, page, D, seed + 2) if cache is None else cache
    n = [h + (counts[b] if counts is not None else T) for b, h in enumerate(held)]
    if stale is not None:  # every slot that holds no token
        for b in range(B):
            for p in range(width):
                live = min(max(n[b] - p * page, 0), page) if n[b] > held[b] else 0
                for t in (cache.k_codes, cache.v_codes):
                    t.view(torch.uint8)[int(bt[b, p]), :, live:] = stale
    if edit is not None:
        edit(cache, bt)
    q = torch.randn(B, T, H, D, generator=_gen(seed), device="cuda") * sharp
    q = q.bfloat16()
    if strided:
        q = q.permute(2, 0, 3, 1).contiguous().permute(1, 3, 0, 2)
    out = kvcache.attend(q, cache, bt, _i32(held), _i32(counts) if counts is not None else None, scale)
    assert out.shape == (B, T, H, D) and out.dtype == torch.bfloat16
    sm = 1 / math.sqrt(D) if scale is None else scale
    for b in range(B):
        c = n[b] - held[b]
        assert not bool(out[b, c:].any())
        if c == 0:
            continue
        ids = bt[b, :-(-n[b] // page)].long()
        for h in range(Hkv):
            k, v = ((x[:, h].view(torch.uint8)[ids].view(E4M3).double() * s[ids, h, None, None].double())
                    .reshape(-1, D)[:n[b]] for x, s in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)))
            want, mag = attention(q[b, :c, h * G:(h + 1) * G].double(), k, v, held[b], sm)
            check_close(out[b, :c, h * G:(h + 1) * G], want, mag * 2.0 ** -10 + want.abs() * 2.0 ** -8)
    return out


@pytest.mark.parametrize("D,page", [(128, 64), (128, 32), (128, 128), (64, 32), (64, 64), (64, 128)])
@pytest.mark.parametrize("Hkv,G", [(2, 4), (1, 1), (3, 8), (1, 16), (2, 5)])
def test_attend_lengths(D, page, Hkv, G):
    held = [0, 1, 31, 32, page - 1, page, 200, 1500]
    _check_attend(8, 1, Hkv, G, D, page, held, seed=G, stale=0x7F)


@pytest.mark.parametrize("T,G", [(2, 4), (3, 3), (8, 1), (9, 1), (5, 7), (33, 2), (17, 8)])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_several_tokens(T, G, D):
    """Causal among the new tokens; unequal counts; rows past counts are 0."""
    _check_attend(5, T, 2, G, D, 32, [0, 30, 64, 700, 5], [T, T, T - 1, T, 0], seed=T * G, stale=0x7F)


@pytest.mark.parametrize("B,held", [(1, 5000), (1, 40000), (2, 20011)])
def test_attend_long(B, held):
    """Keys cut into chunks that are joined, more than once on one stream."""
    for seed in range(2):
        _check_attend(B, 1, 2, 4, 128, 64, [held - 3 * b for b in range(B)], seed=seed, stale=0x7F)
    _check_attend(B, 6, 1, 8, 64, 32, [held - 77 * b for b in range(B)], seed=3)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(1, 1), (1, 2), (1, 3), (1, 5), (1, 8), (3, 4), (5, 4)])
def test_attend_many_pieces(D, T, G):
    """One head over all SMs: joins of more pieces than travel at once, for
    every number of groups that share a row, and for several row tiles."""
    _check_attend(1, T, 1, G, D, 128, [70001], seed=T * G)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hkv,top", [(8, 32, 700), (40, 7, 900), (24, 16, 200), (60, 5, 1500), (300, 1, 600)])
def test_attend_cuts(D, B, Hkv, top):
    """About a head per CTA, and more of them: cuts at heads' ends, within
    heads, and within none, for equal and unequal lengths."""
    _check_attend(B, 1, Hkv, 1, D, 64, [top] * B, seed=B)
    _check_attend(B, 1, Hkv, 2, D, 64, [(i * 7919) % top if i % 5 else 0 for i in range(B)], seed=B + 1)


def test_attend_empty_sequences():
    """No key at all, no new token, and both beside ordinary sequences."""
    _check_attend(4, 1, 2, 4, 128, 64, [0, 300, 0, 64], [0, 1, 1, 0], seed=1, stale=0xFF)
    from voyager_b200 import kvcache

    cache = _cache(2, 2, 64, 128, 0)
    q = torch.randn(0, 1, 4, 128, device="cuda").bfloat16()
    assert kvcache.attend(q, cache, _i32([]).view(0, 1), _i32([])).shape == (0, 1, 4, 128)
    q = torch.randn(3, 0, 4, 128, device="cuda").bfloat16()
    assert kvcache.attend(q, cache, _i32([[0]] * 3), _i32([0] * 3)).shape == (3, 0, 4, 128)


def test_attend_sharp_and_scaled():
    """Large scores (one key takes all), flat ones, negative scale, strides."""
    _check_attend(2, 1, 2, 4, 128, 64, [900, 77], seed=2, sharp=8.0)
    _check_attend(2, 1, 2, 4, 128, 64, [900, 77], seed=3, sharp=1e-6)
    _check_attend(2, 2, 2, 4, 64, 64, [900, 77], seed=4, scale=-0.05, strided=True)


def test_attend_scales_of_any_size():
    """Blocks whose scales lie 2^60 apart, and scales that are no power of two."""
    def far(cache, bt):
        cache.v_scale.copy_(torch.exp2(torch.randint(-60, 0, cache.v_scale.shape, device="cuda").float()))
        cache.k_scale.mul_(1.37)

    _check_attend(3, 1, 2, 4, 128, 32, [500, 1000, 64], seed=5, edit=far)


def test_attend_nan_values():
    """A NaN reaches the rows that see it, and no other: not through a slot past
    the end, nor through a newer token that a row may not see."""
    def nan_at(pos, what):
        def edit(cache, bt):
            getattr(cache, what + "_codes").view(torch.uint8)[int(bt[0, pos // 32]), 0, pos % 32, 3] = 0x7F
        return edit

    for D in (64, 128):
        for what in "kv":
            out = _check_attend(1, 4, 1, 4, D, 32, [61], seed=6, edit=nan_at(63, what))
            assert not bool(out[0, :2].isnan().any()) and bool(out[0, 2:].isnan().any())
            out = _check_attend(1, 4, 1, 4, D, 32, [61], seed=7, edit=nan_at(5, what))
            assert bool(out[0].isnan().any())


def test_attend_offsets_past_32_bits():
    """Pages beyond 2^31 bytes of the cache."""
    from voyager_b200 import kvcache

    pages, Hkv, page, D = 18000, 8, 128, 128
    cache = kvcache.KVCache.empty(pages, Hkv, D, page)
    bt = _i32([[pages - 1, 17, pages - 3], [pages - 2, pages - 4, 3]])
    g = _gen(8)
    for t in (cache.k_codes, cache.v_codes):
        for p in bt.flatten().tolist():
            t[p] = (torch.randn(Hkv, page, D, generator=g, device="cuda") * 50).to(E4M3)
    _check_attend(2, 1, Hkv, 4, D, page, [300, 383], cache=cache, bt=bt, seed=9)
    k = torch.randn(2, 1, Hkv, D, generator=g, device="cuda").bfloat16()
    kvcache.rope_append(k, k, k, kvcache.rotary_table(384, D), cache, bt, _i32([310, 383]))
    assert bool(cache.v_codes[pages - 3, :, 310 - 256].float().any())
    assert bool(cache.k_codes[3, :, 127].float().any())


def test_attend_streams_and_graphs():
    """Calls on two streams do not share their joins; a captured call replays."""
    from voyager_b200 import kvcache

    bt = _table(1, 160, 1)
    cache = _cache(200, 2, 64, 128, 2)
    qs = [torch.randn(1, 1, 8, 128, generator=_gen(i), device="cuda").bfloat16() for i in range(2)]
    held = _i32([10000])
    want = [kvcache.attend(q, cache, bt, held) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kvcache.attend(qs[i], cache, bt, held))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])  # whatever finished first
    q = qs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kvcache.attend(q, cache, bt, held)
    for i in (1, 0):
        q.copy_(qs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])


def test_refusals():
    from voyager_b200 import kvcache

    cache = kvcache.KVCache.empty(4, 2, 128, 64)
    q = torch.zeros(1, 1, 4, 128, device="cuda").bfloat16()
    k = torch.zeros(1, 1, 2, 128, device="cuda").bfloat16()
    tab, bt, held = kvcache.rotary_table(128, 128), _i32([[0, 1]]), _i32([0])
    kvcache.rope_append(q, k, k, tab, cache, bt, held)
    for args in ((q.half(), k, k, tab), (q, k.float(), k, tab)):
        with pytest.raises(NotImplementedError):
            kvcache.rope_append(*args, cache, bt, held)
    for args in ((q[..., :64], k, k, tab), (q[:, :, :3], k, k, tab), (q, k, k[:, :0], tab), (q, k, k, tab[:64]),
                 (q, k, k, tab.double()), (q, k, k, tab[:, :4].contiguous())):
        with pytest.raises(ValueError):
            kvcache.rope_append(*args, cache, bt, held)
    for plan in ((bt.long(), held), (bt, _i32([0, 0])), (bt, held, _i32([[1]])), (bt, held.cpu())):
        with pytest.raises(ValueError):
            kvcache.rope_append(q, k, k, tab, cache, *plan)
        with pytest.raises(ValueError):
            kvcache.attend(q, cache, *plan)
    none = kvcache.KVCache(*(t[:, :0] for t in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)))
    with pytest.raises(ValueError):
        kvcache.rope_append(q, k[:, :, :0], k[:, :, :0], tab, none, bt, held)
    with pytest.raises(ValueError):
        kvcache.attend(q, none, bt, held)
    with pytest.raises(NotImplementedError):
        kvcache.attend(q.float(), cache, bt, held)
    with pytest.raises(ValueError):
        kvcache.attend(q[:, :, :3], cache, bt, held)
    with pytest.raises(ValueError):
        kvcache.KVCache.empty(4, 2, 96)
    bad = kvcache.KVCache(cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale[:2])
    with pytest.raises(ValueError):
        kvcache.attend(q, bad, bt, held)
