"""The cache in 4 bits: the append and the attention over it, and the norms of
query and key heads into either cache, against the formulas in 64 bits.

Tolerances.  Rotation: two float32 products and a sum, 3 * 2^-24 of |a| + |b|.
A norm: a float32 sum of D squares in a tree of at most 16 + 3 additions (its
relative error at most 20 * 2^-24, half of that after the root), rsqrt (2 ulp),
two products: 16 * 2^-24 of the normalised value covers them.  A query must be
the rounding of a value within that of the exact one; a scale the E4M3 rounding
of a quotient within it (and 2^-22 for the division and the factor's product);
a code, given the scale that was stored, the E2M1 rounding of a quotient within
it.  Attention: weights are held in f16 (2^-11 relative), scores are float32
sums of f16 products (below 2^-13 of a weight at these sizes), so an output is
within 2^-10 of sum_j p_j |v_j|, and one bf16 rounding (2^-8).  The weights'
f16 has a floor: the largest weight is at least 2^7 in it (2^15 with up to 16
rows a kv head), its subnormals are 2^-24 apart, so a weight is off by at most
2^-25 there, 2^-32 (2^-40) of the largest, which the division by the weights'
sum does not enlarge: 2^-32 (2^-40) of sum_j |v_j| more.  Codes of 0 are common,
so that columns whose large weights all meet zeros show it."""

import math

import pytest
import torch

from _e4m3_ref import E4M3, attention, check_close, check_rounded, e4m3, pow2_scale, rotate
from _fp4_ref import BLOCK, block_scale, codes_of, e2m1, head_norm, values_of

pytestmark = pytest.mark.gpu
EPS = 1e-6


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


def _table(B, width, seed, extra=2):
    g = _gen(seed)
    return torch.randperm(B * width + extra, generator=g, device="cuda")[:B * width].reshape(B, width).int().contiguous()


def _cache(pages, Hkv, page, D, seed, ones=False):
    """Random codes, scales from 2^-3 to 2^3 with all mantissas, random factors (or 1)."""
    from voyager_b200 import kvcache

    g = _gen(seed)
    f = [None if ones else 0.01 + torch.rand(Hkv, generator=g, device="cuda") for _ in range(2)]
    c = kvcache.KVCache4.empty(pages, Hkv, D, page, k_factor=f[0], v_factor=f[1])
    for t, s in ((c.k_codes, c.k_scale), (c.v_codes, c.v_scale)):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device="cuda"))
        s.view(torch.uint8).copy_(torch.randint(0x20, 0x50, s.shape, generator=g, device="cuda"))
    return c


def _state(c):
    return [t.view(torch.uint8).clone() for t in (c.k_codes, c.v_codes, c.k_scale, c.v_scale)]


def _size(x):
    """The largest finite magnitude of each head: what bounds a rounding.  A pair
    with an infinity is an infinity or NaN whatever the rounding."""
    return torch.where(x.isfinite(), x.abs(), 0.0).amax(-1, keepdim=True)


# ---------------------------------------------------------------------------
def _check_append(B, T, Hkv, G, D, page, held, counts, rot, interleaved, dtype=torch.bfloat16, seed=0, norm="",
                  values=None, fused=True, ones=False, eps=EPS):
    """One append against the definition; norm: which of "q" and "k" are normalised."""
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
    w = {n: (1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dtype) if n in norm else None for n in "qk"}
    table = kvcache.rotary_table(width * page, rot, scaling="linear", factor=2.0)
    bt = _table(B, width, seed + 1)
    cache = _cache(B * width + 2, Hkv, page, D, seed + 2, ones)
    was = _state(cache)
    out = kvcache.rope_append(q, k, v, table, cache, bt, _i32(held), _i32(counts) if counts is not None else None,
                              interleaved, q_norm=w["q"], k_norm=w["k"], eps=eps)
    assert out.shape == q.shape and out.dtype == dtype
    rel = (3 + 16 * (len(norm) > 0)) * 2.0 ** -24
    untouched = [torch.ones_like(t, dtype=torch.bool) for t in was]
    for b in range(B):
        h, n = held[b], counts[b] if counts is not None else T
        assert not bool(out[b, n:].any())
        if n == 0:
            continue
        pos = torch.arange(h, h + n, device="cuda")
        xq, xk = (head_norm(t[b, :n].double(), w[m], eps) for m, t in (("q", q), ("k", k)))
        check_rounded(out[b, :n], rotate(xq, table, pos, interleaved), _size(xq) * 2 * rel)
        pid, slot = bt[b, pos // page].long(), pos % page
        for i, (x, err, f) in enumerate(((rotate(xk, table, pos, interleaved), _size(xk) * 2 * rel, cache.k_factor),
                                         (v[b, :n].double(), None, cache.v_factor))):
            f = f.double()[:, None]
            err = torch.zeros_like(x[..., :1]) if err is None else err
            codes = codes_of((cache.k_codes, cache.v_codes)[i][pid, :, slot]).unflatten(-1, (-1, BLOCK))
            scale = (cache.k_scale, cache.v_scale)[i].view(torch.uint8)[pid, :, slot].view(E4M3).double()
            x = x.unflatten(-1, (-1, BLOCK))
            top = x.abs().amax(-1)
            top = torch.where(x.isnan().any(-1), math.nan, top)
            e22 = 2.0 ** -22 if not ones or i == 0 else 0.0
            lo, hi = (block_scale((top + s * err) * (1 + s * e22), f) for s in (-1, 1))
            fine = (scale >= lo) & (scale <= hi) | lo.isnan() & scale.isnan()
            assert bool(fine.all()), (scale[~fine][:4], lo[~fine][:4], hi[~fine][:4])
            quo = x / (scale * f)[..., None]
            tol = (err / (scale * f))[..., None] + quo.abs() * e22
            tol = torch.where(quo.isinf(), 0.0, tol)  # an infinity saturates exactly
            good = (codes >= e2m1(quo - tol)) & (codes <= e2m1(quo + tol)) | scale.isnan()[..., None]
            assert bool(good.all()), (codes[~good][:4], quo[~good][:4])
            untouched[i][pid, :, slot] = False
            untouched[2 + i][pid, :, slot] = False
    for keep, old, now in zip(untouched, was, _state(cache)):
        assert torch.equal(old[keep], now[keep])
    return cache


@pytest.mark.parametrize("norm", ["", "qk"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot,page", [(128, 128, 64), (128, 32, 128), (64, 64, 32), (64, 16, 64), (128, 96, 32),
                                        (64, 48, 128), (128, 112, 64), (128, 16, 32), (128, 80, 64)])
def test_append4_single_tokens(D, rot, page, interleaved, norm):
    held = [0, 1, page - 1, page, 3 * page + 5]
    _check_append(5, 1, 2, 3, D, page, held, None, rot, interleaved, seed=D + rot, norm=norm)
    _check_append(5, 1, 2, 3, D, page, held, [1, 0, 1, 1, 0], rot, interleaved, torch.float32, seed=D + page, norm=norm)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,page,D", [(2, 32, 64), (31, 32, 128), (33, 32, 128), (64, 64, 64), (130, 64, 128),
                                      (257, 128, 128), (200, 128, 64)])
def test_append4_prompts(T, page, D, dtype):
    """Prompts over several pages, from every kind of start, of unequal counts."""
    _check_append(4, T, 2, 1, D, page, [0, 7, page - 1, 2 * page], [T, T - 1, T, T // 2], D, False, dtype, seed=T,
                  norm="k")
    _check_append(2, T, 1, 2, D, page, [5, 0], None, D // 2, True, dtype, seed=T + 1, fused=False, norm="q")


@pytest.mark.parametrize("D,Hkv,G,rot,interleaved", [(128, 4, 5, 128, False), (64, 7, 1, 48, False), (64, 3, 4, 64, True),
                                                     (128, 32, 1, 112, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append4_many_tokens(D, Hkv, G, rot, interleaved, dtype):
    """More heads and tokens than CTAs at once: several heads a thread, odd counts of them."""
    _check_append(3, 700, Hkv, G, D, 64, [3, 64, 0], [700, 699, 350], rot, interleaved, dtype, seed=D + Hkv, norm="qk")
    _check_append(3, 700, Hkv, G, D, 64, [3, 64, 0], None, rot, interleaved, dtype, seed=D + Hkv)


def test_append4_ties():
    """Quotients exactly between two codes go to the even one: every tie times
    every scale's mantissa, as bfloat16 values with a factor of 1 and of 1/4."""
    from voyager_b200 import kvcache

    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 0.5])
    scales = torch.tensor([m / 8 * 2.0 ** e for e in range(-6, 8) for m in range(8, 16)])
    for f in (1.0, 0.25):
        x = (ties * scales[:, None] * f).repeat(1, 8)[:, None, None].expand(-1, 1, 1, 128).contiguous().cuda()
        assert torch.equal(x.bfloat16().float(), x)
        n = len(scales)
        cache = kvcache.KVCache4.empty(n, 1, 128, 32, k_factor=torch.full((1,), f, device="cuda"),
                                       v_factor=torch.full((1,), f, device="cuda"))
        bt, zero = torch.arange(n, device="cuda").int()[:, None].contiguous(), torch.zeros(n, dtype=torch.int32, device="cuda")
        table = kvcache.rotary_table(32, 128)  # position 0 does not turn
        for dt in (torch.bfloat16, torch.float32):
            kvcache.rope_append(x.to(dt), x.to(dt), x.to(dt), table, cache, bt, zero)
            for codes, scale in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)):
                assert torch.equal(scale[:, 0, 0].float(), scales.cuda()[:, None].expand(-1, 8))
                assert torch.equal(codes_of(codes[:, 0, 0]), e2m1(ties.double().cuda()).repeat(8).expand(n, -1))


def test_append4_specials():
    """Zeros, values beyond the largest scale and below the least, infinities, NaN."""
    def special(x):
        x[0] = 0.0
        x[1] *= 1e5
        x[2] *= 1e-5
        x[3, 0, -1, 5] = float("inf")    # v
        x[3, 1, -1, 40] = float("-inf")
        x[3, 2, -1, 70] = float("nan")
        x[4] *= 1e38

    c = _check_append(5, 3, 2, 1, 128, 64, [9, 70, 3, 62, 0], None, 128, False, seed=3, values=special, ones=True)
    assert int(c.v_scale.float().isnan().sum()) == 1


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("power", [-100, -30, -12, 0, 12, 100])
def test_append4_saturates_under_any_factor(power, tokens):
    """Infinities and the largest values saturate, and ordinary ones keep their codes, whatever the
    factor; every quotient is a power of two's multiple that float32 holds, so nothing is rounded."""
    from voyager_b200 import kvcache

    f, top = 2.0 ** power, torch.finfo(torch.float32).max
    rows = torch.tensor([[math.inf, 1.0, -1.0], [-math.inf, 0.0, top], [-top, top, 0.0], [6 * 448 * f, -448 * f, 0.0],
                         [-6 * f, 5 * f, 1.25 * f], [6e4 * f, 448 * f, -224 * f]], device="cuda")
    n = len(rows)
    x = torch.zeros(n, tokens, 40, 128, device="cuda")
    x[..., 16:19] = rows[:, None, None]
    factor = torch.full((40,), f, device="cuda")
    cache = kvcache.KVCache4.empty(n, 40, 128, 64, k_factor=factor, v_factor=factor)
    bt = torch.arange(n, device="cuda").int()[:, None].contiguous()
    held = torch.zeros(n, dtype=torch.int32, device="cuda")
    table = kvcache.rotary_table(64, 16)  # columns from 16 on do not turn
    kvcache.rope_append(x, x, x, table, cache, bt, held)
    y = x[0:, :, 0, 16:32].double()
    scale = block_scale(y.abs().amax(-1), f)
    want = e2m1(y / (scale * f)[..., None])
    for codes, scales in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)):
        got = codes_of(codes[:, :, :tokens].transpose(1, 2)).unflatten(-1, (8, 16))[..., 1, :]
        assert torch.equal(scales.float()[:, :, :tokens, 1].transpose(1, 2).double(), scale[..., None].expand(-1, -1, 40))
        assert torch.equal(got, want[:, :, None].expand_as(got))


def test_append4_token_by_token_is_the_prompt():
    """Tokens do not touch each other's blocks: one at a time, in pieces and at
    once give the same bytes."""
    from voyager_b200 import kvcache

    g = _gen(5)
    T, Hkv, G, D, page = 150, 2, 2, 128, 64
    x = torch.randn(1, T, (G + 2) * Hkv, D, generator=g, device="cuda").bfloat16()
    q, k, v = x.split([G * Hkv, Hkv, Hkv], 2)
    w = torch.rand(D, generator=g, device="cuda").bfloat16() + 0.5
    table, bt = kvcache.rotary_table(192, D), _i32([[2, 0, 1]])
    states = []
    for step in (1, 7, T):
        c = kvcache.KVCache4.empty(3, Hkv, D, page)
        out = [kvcache.rope_append(q[:, t:t + step], k[:, t:t + step], v[:, t:t + step], table, c, bt, _i32([t]),
                                   q_norm=w, k_norm=w) for t in range(0, T, step)]
        states.append([torch.cat(out, 1)] + _state(c))
    for s in states[1:]:
        assert all(torch.equal(a, b) for a, b in zip(states[0], s))


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,rot,page,interleaved", [(128, 128, 64, False), (64, 32, 32, True), (128, 96, 128, False)])
@pytest.mark.parametrize("B,T", [(5, 1), (3, 3), (4, 40), (3, 300)])
def test_norm_append_e4m3(B, T, D, rot, page, interleaved, dtype):
    """Normalised heads into the E4M3 cache: the same blocks as an append of heads
    that were normalised before, up to the norm's own error."""
    from voyager_b200 import kvcache

    g = _gen(B * T + D)
    Hkv, G = 2, 3
    held = [(37 * b) % (2 * page) for b in range(B)]
    counts = [T - b % 2 * (T // 2) for b in range(B)]
    width = -(-(2 * page + T) // page)
    qkv = (torch.randn(B, T, Hkv * (G + 2), D, generator=g, device="cuda") * 3).to(dtype)
    q, k, v = qkv.split([Hkv * G, Hkv, Hkv], 2)
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2))
    table = kvcache.rotary_table(width * page, rot)
    bt = _table(B, width, 1)
    cache = kvcache.KVCache.empty(B * width + 2, Hkv, D, page)
    out = kvcache.rope_append(q, k, v, table, cache, bt, _i32(held), _i32(counts), interleaved, q_norm=wq, k_norm=wk)
    plain = kvcache.KVCache.empty(B * width + 2, Hkv, D, page)
    kvcache.rope_append(q, k, v, table, plain, bt, _i32(held), _i32(counts), interleaved)
    assert torch.equal(plain.v_codes.view(torch.uint8), cache.v_codes.view(torch.uint8))
    assert torch.equal(plain.v_scale, cache.v_scale)
    rel = 19 * 2.0 ** -24
    for b in range(B):
        h, n = held[b], counts[b]
        assert not bool(out[b, n:].any())
        if not n:
            continue
        pos = torch.arange(h, h + n, device="cuda")
        xq, xk = head_norm(q[b, :n].double(), wq, EPS), head_norm(k[b, :n].double(), wk, EPS)
        check_rounded(out[b, :n], rotate(xq, table, pos, interleaved), xq.abs().amax(-1, keepdim=True) * 2 * rel)
        x, err = rotate(xk, table, pos, interleaved), xk.abs().amax(-1, keepdim=True) * 2 * rel
        for p in range(h // page, (h + n - 1) // page + 1):
            lo, hi, pid = max(h, p * page), min(h + n, (p + 1) * page), int(bt[b, p])
            for hd in range(Hkv):
                y, e = x[lo - h:hi - h, hd], err[lo - h:hi - h, hd]
                s, top = float(cache.k_scale[pid, hd]), float(y.abs().max())
                fresh = 1.0 if lo > p * page else 0.0  # empty caches have scales of 1
                assert s in {max(pow2_scale(top * (1 + d)), fresh) for d in (-1e-5, 0.0, 1e-5)}
                c = cache.k_codes[pid, hd, lo - p * page:hi - p * page].double()
                assert bool(((c >= e4m3((y - e) / s)) & (c <= e4m3((y + e) / s))).all())


def test_norm_of_one_side_and_eps():
    """A norm of the queries alone, of the keys alone, and an eps that weighs."""
    for norm in ("q", "k", "qk"):
        _check_append(3, 2, 2, 2, 64, 32, [0, 31, 50], None, 64, False, norm=norm, eps=0.7, seed=1)
        _check_append(3, 90, 2, 8, 128, 32, [0, 31, 50], None, 64, False, norm=norm, eps=0.7, seed=2)


def test_norm_of_zero_heads():
    """A head of zeros stays zero (eps keeps the factor finite)."""
    def zero(x):
        x[0] = 0.0

    _check_append(2, 3, 2, 2, 128, 64, [0, 9], None, 128, False, norm="qk", values=zero, seed=6)


# ---------------------------------------------------------------------------
def test_unpack():
    from voyager_b200 import kvcache

    for pages, Hkv, page, D in ((5, 3, 32, 64), (1, 1, 128, 128), (300, 8, 64, 128), (0, 2, 32, 64)):
        c = _cache(pages, Hkv, page, D, pages)
        got = kvcache.unpack(c)
        for t, raw in zip(got, (c.k_codes, c.v_codes)):
            assert t.dtype == E4M3 and t.shape == (pages, Hkv, page, D)
            assert torch.equal(t.double(), codes_of(raw))


# ---------------------------------------------------------------------------
def _bound(want, mag, v, rows):
    floor = 2.0 ** (-40 if rows <= 16 else -32)
    return mag * 2.0 ** -10 + want.abs() * 2.0 ** -8 + floor * v.nan_to_num(0.0).abs().sum(0)


def _check_attend(B, T, Hkv, G, D, page, held, counts=None, seed=0, scale=None, stale=True, cache=None, bt=None,
                  sharp=1.0, edit=None, strided=False):
    from voyager_b200 import kvcache

    H = Hkv * G
    width = max(1, -(-max(h + T for h in held) // page))
    bt = _table(B, width, seed + 1) if bt is None else bt
    cache = _cache(int(bt.max()) + 2, Hkv, page, D, seed + 2) if cache is None else cache
    n = [h + (counts[b] if counts is not None else T) for b, h in enumerate(held)]
    if stale:  # every slot that holds no token: scales of NaN
        for b in range(B):
            for p in range(width):
                live = min(max(n[b] - p * page, 0), page) if n[b] > held[b] else 0
                for t in (cache.k_scale, cache.v_scale):
                    t.view(torch.uint8)[int(bt[b, p]), :, live:] = 0x7F
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
            k, v = (values_of(x[ids, h], s.view(torch.uint8)[ids, h].view(E4M3), f[h].double()).reshape(-1, D)[:n[b]]
                    for x, s, f in ((cache.k_codes, cache.k_scale, cache.k_factor),
                                    (cache.v_codes, cache.v_scale, cache.v_factor)))
            want, mag = attention(q[b, :c, h * G:(h + 1) * G].double(), k, v, held[b], sm)
            check_close(out[b, :c, h * G:(h + 1) * G], want, _bound(want, mag, v, T * G))
    return out


@pytest.mark.parametrize("D,page", [(128, 64), (128, 32), (128, 128), (64, 32), (64, 64), (64, 128)])
@pytest.mark.parametrize("Hkv,G", [(2, 4), (1, 1), (3, 8), (1, 16), (2, 5), (1, 24)])
def test_attend4_lengths(D, page, Hkv, G):
    held = [0, 1, 31, 32, page - 1, page, 200, 1500]
    _check_attend(8, 1, Hkv, G, D, page, held, seed=G)


@pytest.mark.parametrize("T,G", [(2, 4), (3, 3), (8, 1), (9, 1), (5, 7), (33, 2), (17, 8), (128, 1), (129, 1), (70, 4),
                                 (257, 1), (19, 27)])
@pytest.mark.parametrize("D", [64, 128])
def test_attend4_several_tokens(T, G, D):
    """Causal among the new tokens; unequal counts; rows past counts are 0."""
    _check_attend(5, T, 2, G, D, 32, [0, 30, 64, 700, 5], [T, T, T - 1, T, 0], seed=T * G)


@pytest.mark.parametrize("B,held", [(1, 5000), (1, 40000), (2, 20011)])
def test_attend4_long(B, held):
    """Keys cut into chunks that are joined, more than once on one stream."""
    for seed in range(2):
        _check_attend(B, 1, 2, 4, 128, 64, [held - 3 * b for b in range(B)], seed=seed)
    _check_attend(B, 6, 1, 8, 64, 32, [held - 77 * b for b in range(B)], seed=3)
    _check_attend(B, 40, 1, 5, 128, 64, [held - 77 * b for b in range(B)], seed=4)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(1, 1), (1, 3), (1, 8), (3, 4), (5, 4), (40, 4)])
def test_attend4_many_pieces(D, T, G):
    """One head over all SMs."""
    _check_attend(1, T, 1, G, D, 128, [70001], seed=T * G)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hkv,top", [(8, 32, 700), (40, 7, 900), (60, 5, 1500), (300, 1, 600)])
def test_attend4_cuts(D, B, Hkv, top):
    """About a head per CTA, and more of them, for equal and unequal lengths."""
    _check_attend(B, 1, Hkv, 1, D, 64, [top] * B, seed=B)
    _check_attend(B, 1, Hkv, 2, D, 64, [(i * 7919) % top if i % 5 else 0 for i in range(B)], seed=B + 1)


@pytest.mark.parametrize("D,Hkv,G,page", [(128, 2, 4, 64), (64, 1, 5, 32), (128, 1, 1, 128), (64, 2, 8, 64)])
def test_attend4_prompts(D, Hkv, G, page):
    """Prompts over themselves and over what the cache holds: many tiles of rows,
    rows whose first tile of keys is all there is, odd ends everywhere."""
    _check_attend(2, 600, Hkv, G, D, page, [0, 0], [600, 411], seed=1)
    _check_attend(2, 300, Hkv, G, D, page, [1000, 77], seed=2)
    _check_attend(1, 513, Hkv, G, D, page, [127], seed=3)


@pytest.mark.parametrize("B,T,Hkv,G,D", [(40, 130, 4, 2, 128), (200, 70, 2, 2, 64), (75, 129, 2, 2, 64), (3, 1100, 8, 4, 64)])
def test_attend4_many_heads(B, T, Hkv, G, D):
    """More row tiles than CTAs, of equal and of unequal sizes, some of them empty;
    more sequences than a CTA keeps plans of."""
    held = [(i * 37) % 150 for i in range(B)]
    counts = [0 if i % 7 == 3 else T - (i * 29) % T for i in range(B)]
    _check_attend(B, T, Hkv, G, D, 64, held, counts, seed=B)
    _check_attend(B, T, Hkv, G, D, 64, [100] * B, seed=B + 1)


@pytest.mark.parametrize("T,G", [(1, 4), (3, 8), (9, 8), (60, 4)])
@pytest.mark.parametrize("D", [64, 128])
def test_attend4_growing_scores(T, G, D):
    """Keys that grow along the sequence: the running maximum moves on and on."""
    def grow(cache, bt):
        raw = cache.k_scale.view(torch.uint8)
        pos = torch.arange(bt.shape[1] * 32, device="cuda").view(-1, 32)
        for p in range(bt.shape[1]):
            raw[int(bt[0, p])] = (0x10 + pos[p] * 0x30 // pos.numel()).byte()[None, :, None]
        cache.k_factor.fill_(0.2)

    _check_attend(1, T, 2, G, D, 32, [2500], seed=11, edit=grow, stale=False)


@pytest.mark.parametrize("T,G", [(2, 4), (40, 4), (90, 2)])
def test_attend4_queries_that_are_no_numbers(T, G):
    """A NaN or an infinity in a query stays in its row."""
    from voyager_b200 import kvcache

    bt, cache = _table(1, 16, 1), _cache(20, 2, 64, 128, 2)
    q = torch.randn(1, T, 2 * G, 128, generator=_gen(3), device="cuda").bfloat16()
    want = kvcache.attend(q, cache, bt, _i32([800]))
    for bad in (float("nan"), float("inf")):
        x = q.clone()
        x[0, 1, 1, 7] = bad
        out = kvcache.attend(x, cache, bt, _i32([800]))
        assert bool(out[0, 1, 1].isnan().all())
        keep = torch.ones(1, T, 2 * G, dtype=torch.bool, device="cuda")
        keep[0, 1, 1] = False
        assert torch.equal(out[keep], want[keep])


def test_attend4_kernels_take_turns():
    """Calls of few and of many rows on one stream, and captured together, share
    their counters and leave them as they were."""
    from voyager_b200 import kvcache

    bt = _table(6, 70, 1)
    cache = _cache(430, 4, 64, 128, 2)
    held = _i32([4000, 10, 900, 0, 2000, 333])
    qs = [torch.randn(6, T, 16, 128, generator=_gen(T), device="cuda").bfloat16() for T in (1, 200, 4, 60, 12)]
    want = [kvcache.attend(q, cache, bt, held) for q in qs]
    for _ in range(4):
        assert all(torch.equal(kvcache.attend(q, cache, bt, held), w) for q, w in zip(qs, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [kvcache.attend(q, cache, bt, held) for q in qs]
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_attend4_empty_sequences():
    """No key at all, no new token, and both beside ordinary sequences."""
    from voyager_b200 import kvcache

    _check_attend(4, 1, 2, 4, 128, 64, [0, 300, 0, 64], [0, 1, 1, 0], seed=1)
    _check_attend(4, 200, 2, 4, 128, 64, [0, 300, 0, 64], [0, 1, 200, 0], seed=1)
    cache = _cache(2, 2, 64, 128, 0)
    for T in (1, 50):
        q = torch.randn(0, T, 4, 128, device="cuda").bfloat16()
        assert kvcache.attend(q, cache, _i32([]).view(0, 1), _i32([])).shape == (0, T, 4, 128)
    q = torch.randn(3, 0, 4, 128, device="cuda").bfloat16()
    assert kvcache.attend(q, cache, _i32([[0]] * 3), _i32([0] * 3)).shape == (3, 0, 4, 128)


@pytest.mark.parametrize("T", [1, 2, 60])
def test_attend4_sharp_and_scaled(T):
    """Large scores (one key takes all), flat ones, negative scale, strides."""
    _check_attend(2, T, 2, 4, 128, 64, [900, 77], seed=2, sharp=8.0)
    _check_attend(2, T, 2, 4, 128, 64, [900, 77], seed=3, sharp=1e-6)
    _check_attend(2, T, 2, 4, 64, 64, [900, 77], seed=4, scale=-0.05, strided=True)


@pytest.mark.parametrize("T", [1, 60])
def test_attend4_scales_and_factors_of_any_size(T):
    """All of E4M3's range of scales, and factors far from 1."""
    def far(cache, bt):
        for s in (cache.k_scale, cache.v_scale):
            raw = s.view(torch.uint8)
            raw.copy_(torch.where(raw == 0x7F, raw, torch.randint(1, 0x7F, raw.shape, generator=_gen(9), device="cuda").byte()))
        cache.k_factor.copy_(torch.tensor([1e-3, 3e-4]))
        cache.v_factor.copy_(torch.tensor([1e-20, 1e20]))

    _check_attend(3, T, 2, 4, 128, 32, [500, 1000, 64], seed=5, edit=far)
    _check_attend(3, T, 2, 4, 64, 32, [500, 1000, 64], seed=5, edit=far)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(4, 4), (40, 4)])
def test_attend4_nan_values(D, T, G):
    """A NaN reaches the rows that see it, and no other: not through a slot past
    the end, nor through a newer token that a row may not see."""
    def nan_at(pos, what):
        def edit(cache, bt):
            getattr(cache, what + "_scale").view(torch.uint8)[int(bt[0, pos // 32]), 0, pos % 32, 1] = 0x7F
        return edit

    for what in "kv":
        out = _check_attend(1, T, 1, G, D, 32, [61], seed=6, edit=nan_at(63, what))
        assert not bool(out[0, :2].isnan().any()) and bool(out[0, 2:].isnan().any())
        out = _check_attend(1, T, 1, G, D, 32, [61], seed=7, edit=nan_at(5, what))
        assert bool(out[0].isnan().any())


@pytest.mark.parametrize("T", [1, 30])
def test_attend4_offsets_past_32_bits(T):
    """Pages beyond 2^31 bytes of the cache."""
    from voyager_b200 import kvcache

    pages, Hkv, page, D = 36000, 4, 128, 128
    cache = kvcache.KVCache4.empty(pages, Hkv, D, page)
    bt = _i32([[pages - 1, 17, pages - 3], [pages - 2, pages - 4, 3]])
    g = _gen(8)
    for t in (cache.k_codes, cache.v_codes):
        for p in bt.flatten().tolist():
            t[p] = torch.randint(0, 256, t[p].shape, generator=g, device="cuda").byte()
    _check_attend(2, T, Hkv, 4, D, page, [300 - T, 383 - T], cache=cache, bt=bt, seed=9)
    k = torch.randn(2, 1, Hkv, D, generator=g, device="cuda").bfloat16()
    before = cache.v_codes[pages - 3, :, 310 - 256].clone(), cache.k_codes[3, :, 127].clone()
    kvcache.rope_append(k, k, k, kvcache.rotary_table(384, D), cache, bt, _i32([310, 383]))
    assert not torch.equal(before[0], cache.v_codes[pages - 3, :, 310 - 256])
    assert not torch.equal(before[1], cache.k_codes[3, :, 127])


@pytest.mark.parametrize("T,G,D", [(40, 4, 128), (60, 4, 64), (30, 4, 128), (25, 5, 64), (3, 4, 64)])
def test_attend4_many_heads_on_two_streams(T, G, D):
    """Heads taken whole, cut and joined, or few rows: calls on two streams and two graphs at once
    take theirs from counters of their own, and whoever takes a head computes the same."""
    from voyager_b200 import kvcache

    B, Hkv = 40, 8
    bt = _table(B, 7, 1)
    cache = _cache(B * 7 + 2, Hkv, 64, D, 2)
    held = _i32([300 + 2 * b for b in range(B)])
    qs = [torch.randn(B, T, Hkv * G, D, generator=_gen(i), device="cuda").bfloat16() for i in range(2)]
    want = [kvcache.attend(q, cache, bt, held) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kvcache.attend(qs[i], cache, bt, held))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            outs.append(kvcache.attend(qs[i], cache, bt, held))
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    counts = [int(n) for n in torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(1))]
    _check_attend(B, T, Hkv, G, D, 64, held.tolist(), counts, seed=T)


@pytest.mark.parametrize("T", [1, 40])
def test_attend4_streams_and_graphs(T):
    """Calls on two streams do not share their joins; a captured call replays."""
    from voyager_b200 import kvcache

    bt = _table(1, 160, 1)
    cache = _cache(200, 2, 64, 128, 2)
    qs = [torch.randn(1, T, 8, 128, generator=_gen(i), device="cuda").bfloat16() for i in range(2)]
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
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(kvcache.attend(q, cache, bt, held))
    for i in (1, 0):
        q.copy_(qs[i])
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):  # two graphs at once
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[i]) for o in outs)


@pytest.mark.parametrize("T", [1, 5, 40])
@pytest.mark.parametrize("D,page", [(128, 64), (64, 32)])
def test_attend4_leaves_out_pages_outside_the_cache(T, D, page):
    """The keys of a page outside the cache are not seen; the plan is reported."""
    import voyager_b200
    from voyager_b200 import _lib, kvcache

    Hkv, G, held = 2, 4, 6 * page + 3
    bt = _table(1, 8, 3)
    cache = _cache(12, Hkv, page, D, 4)
    for bad in (-1, 12, 2 ** 30):
        bt2 = bt.clone()
        bt2[0, 1] = bt2[0, 4] = bad
        q = torch.randn(1, T, Hkv * G, D, generator=_gen(T), device="cuda").bfloat16()
        out = kvcache.attend(q, cache, bt2, _i32([held]))
        with pytest.raises(_lib.VqError, match="plan"):
            voyager_b200.check_errors()
        n = held + T
        keep = torch.ones(n, dtype=torch.bool, device="cuda")
        for p in (1, 4):
            keep[p * page:(p + 1) * page] = False
        ids = bt[0, :-(-n // page)].long()
        for h in range(Hkv):
            k, v = (values_of(x[ids, h], s.view(torch.uint8)[ids, h].view(E4M3), f[h].double()).reshape(-1, D)[:n][keep]
                    for x, s, f in ((cache.k_codes, cache.k_scale, cache.k_factor),
                                    (cache.v_codes, cache.v_scale, cache.v_factor)))
            want, mag = attention(q[0, :, h * G:(h + 1) * G].double(), k, v, held - 2 * page, 1 / math.sqrt(D))
            check_close(out[0, :, h * G:(h + 1) * G], want, _bound(want, mag, v, T * G))


def test_plan_errors_are_reported():
    """Plans that do not fit leave the tokens out, touch nothing outside and
    set the sticky word."""
    import voyager_b200
    from voyager_b200 import _lib, kvcache

    def go(held, counts, bt, T=2):
        cache = _cache(4, 1, 32, 64, 6)
        before = cache.k_scale.view(torch.uint8).clone().fill_(0)
        cache.k_scale.view(torch.uint8).fill_(0)
        q = torch.ones(1, T, 1, 64, device="cuda").bfloat16()
        kvcache.rope_append(q, q, q, kvcache.rotary_table(64, 64), cache, bt, _i32([held]), _i32([counts]))
        with pytest.raises(_lib.VqError, match="plan"):
            voyager_b200.check_errors()
        for t in (1, 40):
            n = counts if t == 1 else counts + 38
            a = kvcache.attend(q[:, :1].expand(1, t, 1, 64), cache, bt, _i32([held]), _i32([n]))
            with pytest.raises(_lib.VqError, match="plan"):
                voyager_b200.check_errors()
            assert a.shape == (1, t, 1, 64)
        return int((cache.k_scale.view(torch.uint8) != before).any(-1).sum())

    ok = _i32([[1, 2]])
    assert go(-1, 1, ok) == 0
    assert go(3, -42, ok) == 0
    assert go(63, 2, ok) == 1     # one slot left
    assert go(1000, 1, ok) == 0
    assert go(3, 1, _i32([[-1, 2]])) == 0
    assert go(3, 1, _i32([[4, 2]])) == 0


@pytest.mark.parametrize("pages,width", [(3, 0), (0, 0), (0, 2)])
@pytest.mark.parametrize("T", [1, 40])
def test_empty_tables_and_caches(pages, width, T):
    """No page to read: zeros, and the plan is reported where it holds tokens."""
    import voyager_b200
    from voyager_b200 import _lib, kvcache

    cache = kvcache.KVCache4.empty(pages, 2, 64, 32)
    q = torch.randn(2, T, 4, 64, device="cuda").bfloat16()
    bt = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
    k = torch.randn(2, T, 2, 64, device="cuda").bfloat16()
    for counts in (None, _i32([0, 0])):
        kvcache.rope_append(q, k, k, kvcache.rotary_table(64, 64), cache, bt, _i32([0, 0]), counts)
        assert not bool(kvcache.attend(q, cache, bt, _i32([0, 0]), counts).any())
        if counts is None:
            with pytest.raises(_lib.VqError, match="plan"):
                voyager_b200.check_errors()
        else:
            voyager_b200.check_errors()


def test_a_gradient_is_not_lost_in_silence():
    from voyager_b200 import kvcache

    cache = _cache(2, 2, 64, 128, 1)
    k = torch.randn(1, 1, 2, 128, device="cuda").bfloat16()
    w = torch.ones(128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = kvcache.rope_append(k, k, k, kvcache.rotary_table(64, 128), cache, _i32([[0]]), _i32([3]), q_norm=w)
    assert out.requires_grad
    with pytest.raises(Exception, match="rope_append"):
        out.sum().backward()
    for T in (1, 40):
        q = torch.randn(1, T, 4, 128, device="cuda").bfloat16().requires_grad_()
        with pytest.raises(Exception, match="attend"):
            kvcache.attend(q, cache, _i32([[0]]), _i32([3])).sum().backward()


def test_refusals():
    from voyager_b200 import kvcache

    cache = kvcache.KVCache4.empty(4, 2, 128, 64)
    q = torch.zeros(1, 1, 4, 128, device="cuda").bfloat16()
    k = torch.zeros(1, 1, 2, 128, device="cuda").bfloat16()
    w = torch.ones(128, device="cuda").bfloat16()
    tab, bt, held = kvcache.rotary_table(128, 128), _i32([[0, 1]]), _i32([0])
    kvcache.rope_append(q, k, k, tab, cache, bt, held, q_norm=w, k_norm=w)
    shifted = torch.ones(136, device="cuda").bfloat16()[1:129]  # not on 16 bytes: copied
    kvcache.rope_append(q, k, k, tab, cache, bt, held, q_norm=shifted)
    kvcache.rope_append(q, k, k, tab, cache, bt, held, q_norm=w[:1].expand(128))
    for bad in (w.float(), w[:64], w[None], w.cpu()):
        for c in (cache, kvcache.KVCache.empty(4, 2, 128, 64)):
            with pytest.raises(ValueError):
                kvcache.rope_append(q, k, k, tab, c, bt, held, q_norm=bad)
            with pytest.raises(ValueError):
                kvcache.rope_append(q, k, k, tab, c, bt, held, k_norm=bad)
    for args in ((q[..., :64], k, k, tab), (q[:, :, :3], k, k, tab), (q, k, k[:, :0], tab), (q, k, k, tab[:64])):
        with pytest.raises(ValueError):
            kvcache.rope_append(*args, cache, bt, held)

    def but(**kw):
        return kvcache.KVCache4(**{**cache.__dict__, **kw})

    wrong = [but(k_factor=cache.k_factor[:1]), but(v_factor=cache.v_factor.double()), but(k_factor=cache.k_factor.cpu()),
             but(k_scale=cache.k_scale[:2]), but(v_scale=cache.v_scale[..., :4].contiguous()),
             but(k_codes=cache.k_codes[:, :, :32].contiguous()), but(v_codes=cache.v_codes.transpose(0, 1))]
    for c in wrong:
        with pytest.raises(ValueError):
            kvcache.attend(q, c, bt, held)
        with pytest.raises(ValueError):
            kvcache.rope_append(q, k, k, tab, c, bt, held)
        with pytest.raises(ValueError):
            kvcache.unpack(c)
    for c in (but(k_codes=cache.k_codes.view(E4M3)), but(k_scale=cache.k_scale.float())):
        with pytest.raises(NotImplementedError):
            kvcache.attend(q, c, bt, held)
    with pytest.raises(TypeError):
        kvcache.attend(q, but(k_factor=None), bt, held)
    with pytest.raises(NotImplementedError):
        kvcache.attend(q.float(), cache, bt, held)
    with pytest.raises(ValueError):
        kvcache.KVCache4.empty(4, 2, 96)
