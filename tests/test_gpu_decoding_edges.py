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


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("D,T", [(64, 1), (64, 2), (64, 3), (64, 8), (128, 1), (128, 2), (128, 4)])
def test_every_held_code_follows_a_grown_scale(D, T):
    """Few new tokens whose values need larger scales in every block: all the
    codes that a block holds are brought to its new scale, for any number of
    lanes a block, and the scale is the one that the new values need."""
    from voyager_b200 import kvcache

    B, Hkv, page = 150, 3, 64
    cache = _cache(2 * B, Hkv, page, D, D + T)
    old = [t.clone() for t in (cache.k_codes.view(torch.uint8), cache.v_codes.view(torch.uint8), cache.k_scale,
                               cache.v_scale)]
    bt = torch.randperm(2 * B, generator=_gen(6), device="cuda").view(B, 2).int()
    held = torch.randint(1, page - T + 1, (B,), generator=_gen(7), device="cuda").int()  # the new tokens end in page 0
    k, v = (torch.randn(B, T, Hkv, D, generator=_gen(s), device="cuda") for s in (8, 9))
    # keys of +-2^10, values of +-2^4: scales 2^2 and 2^-4, larger than the 2^-9 .. 2^-4 held
    k, v = (k.sign() * 2.0 ** 10).bfloat16(), (v.sign() * 2.0 ** 4).bfloat16()
    one = torch.tensor([1.0, 0.0], device="cuda").expand(2 * page, D // 2, 2).contiguous()  # no rotation
    kvcache.rope_append(k, k, v, one, cache, bt, held)
    pid = bt[:, 0].long()
    for codes, scale, was, s0, new, s1 in ((cache.k_codes, cache.k_scale, old[0], old[2], k, 2.0 ** 2),
                                           (cache.v_codes, cache.v_scale, old[1], old[3], v, 2.0 ** -4)):
        assert bool((scale[pid] == s1).all())
        assert torch.equal(scale[bt[:, 1].long()], s0[bt[:, 1].long()])
        want = (was.view(E4M3)[pid].float() * (s0[pid] / s1)[..., None, None]).to(E4M3)  # a power of two: exact
        for b in range(B):
            h = int(held[b])
            got = codes[pid[b]].float()
            assert torch.equal(got[:, :h], want[b, :, :h].float())
            assert torch.equal(got[:, h:h + T], new[b].transpose(0, 1).float() / s1)
            assert torch.equal(codes.view(torch.uint8)[pid[b], :, h + T:], was[pid[b], :, h + T:])


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("pages,width", [(3, 0), (0, 0), (0, 2)])
def test_empty_tables_and_caches(pages, width):
    """A block table of no columns and a cache of no pages hold no token: rows
    see no key, nothing is written, and only a plan that names tokens is
    reported."""
    import voyager_b200
    from voyager_b200 import _lib, kvcache

    B, T, H, Hkv, D, page = 3, 2, 4, 2, 64, 32
    cache = _cache(pages, Hkv, page, D, 1)
    before = cache.k_codes.view(torch.uint8).clone()
    bt = torch.zeros(B, width, dtype=torch.int32, device="cuda")
    table = kvcache.rotary_table(width * page, D)
    q = torch.ones(B, T, H, D, device="cuda").bfloat16()
    k = torch.ones(B, T, Hkv, D, device="cuda").bfloat16()
    zero = _i32([0] * B)
    turned = kvcache.rope_append(q, k, k, table, cache, bt, zero, zero)
    out = kvcache.attend(q, cache, bt, zero, zero)
    assert turned.shape == out.shape == q.shape and not bool(turned.any()) and not bool(out.any())
    voyager_b200.check_errors()
    kvcache.rope_append(q, k, k, table, cache, bt, zero)
    with pytest.raises(_lib.VqError, match="plan"):
        voyager_b200.check_errors()
    for counts in (None, _i32([0, T, 0]), _i32([0, -1, 0])):
        out = kvcache.attend(q, cache, bt, zero, counts)
        assert not bool(out.any())
        with pytest.raises(_lib.VqError, match="plan"):
            voyager_b200.check_errors()
    assert torch.equal(cache.k_codes.view(torch.uint8), before)


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("C", [120, 136, 392, 1032, 129, 131, 250])
def test_norm_of_a_row_whose_squares_vanish(C):
    """With eps = 0 and squares below float32's range the row's factor is
    infinite: y and the scales are infinities in every block, the last and
    shorter one too, and the codes NaN."""
    from voyager_b200 import fp8block

    x = torch.full((2, C), 1e-30, device="cuda")
    codes, scale, _ = fp8block.rmsnorm_quantize(x, torch.ones(C, device="cuda"), 0.0)
    assert bool((scale == math.inf).all()), scale
    assert bool(codes.float().isnan().all())


# ---------------------------------------------------------------------------
def test_a_gradient_is_not_lost_in_silence():
    """The operators have no derivative: asked for one, the backward pass says
    so.  The values are those without gradients."""
    from voyager_b200 import fp8block, kvcache

    def raises(y):
        assert y.requires_grad
        with pytest.raises(RuntimeError, match="not implemented"):
            y.float().sum().backward()

    x = torch.randn(4, 256, generator=_gen(1), device="cuda")
    w = torch.ones(256, device="cuda")
    plain = fp8block.rmsnorm_quantize(x, w, residual=x)
    assert not any(t.requires_grad for t in plain)
    for args in ((x.clone().requires_grad_(), w, x), (x, w.clone().requires_grad_(), x),
                 (x, w, x.clone().requires_grad_())):
        got = fp8block.rmsnorm_quantize(args[0], args[1], residual=args[2])
        for a, b in zip(got, plain):
            assert torch.equal(a.detach().float(), b.float())
            raises(a)
        with torch.no_grad():
            assert not any(t.requires_grad for t in fp8block.rmsnorm_quantize(args[0], args[1], residual=args[2]))
    raises(fp8block.quantize(x.clone().requires_grad_())[1])
    c, s = fp8block.quantize(x)
    wc, ws = fp8block.quantize_weight(torch.randn(96, 256, generator=_gen(2), device="cuda"))
    bias = torch.zeros(96, device="cuda").bfloat16()
    want = fp8block.linear(c, s, wc, ws, bias)
    for i in (1, 3, 4):
        args = [c, s, wc, ws, bias]
        args[i] = args[i].clone().requires_grad_()
        got = fp8block.linear(*args)
        assert torch.equal(got.detach(), want)
        raises(got)
    qkv = [torch.randn(1, 3, h, 64, generator=_gen(3), device="cuda").bfloat16() for h in (4, 2, 2)]
    table, bt, held = kvcache.rotary_table(64, 64), _i32([[0, 1]]), _i32([0])
    for i in range(3):
        cache = kvcache.KVCache.empty(2, 2, 64, 32)
        args = list(qkv)
        args[i] = args[i].clone().requires_grad_()
        q = kvcache.rope_append(*args, table, cache, bt, held)
        raises(q)
        raises(kvcache.attend(kvcache.rope_append(*args, table, cache, bt, held), cache, bt, held))
    with torch.inference_mode():
        assert not kvcache.attend(qkv[0], cache, bt, held).requires_grad


# ---------------------------------------------------------------------------
def test_calls_on_the_per_thread_default_stream():
    """One handle names a stream of its own in each thread: calls that overlap
    there do not share their joins.  Each thread allocates from a pool of its
    own, as the allocator too knows streams by their handles."""
    import threading

    from voyager_b200 import kvcache

    cache = _cache(500, 1, 64, 128, 2)
    bt = torch.randperm(500, generator=_gen(1), device="cuda").view(1, 500).int()
    qs = [torch.randn(1, 1, 8, 128, generator=_gen(i), device="cuda").bfloat16() for i in range(3)]
    held = _i32([31000])
    want = [kvcache.attend(q, cache, bt, held) for q in qs]
    torch.cuda.synchronize()
    pools, got, errors = [torch.cuda.MemPool() for _ in qs], [[] for _ in qs], []

    def work(i):
        try:
            side = torch.cuda.ExternalStream(2)  # cudaStreamPerThread
            with torch.cuda.use_mem_pool(pools[i]), torch.cuda.stream(side):
                torch.cuda._sleep(10_000_000)
                for _ in range(30):
                    got[i].append(kvcache.attend(qs[i], cache, bt, held))
                side.synchronize()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(qs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for w, outs in zip(want, got):
        assert len(outs) == 30 and all(torch.equal(o, w) for o in outs)


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("C", [12288, 16384])
def test_norm_many_wide_rows(C, dtype):
    """More rows than CTAs where a row takes a CTA's whole width."""
    from test_gpu_fp8block import _check_norm

    g = _gen(C)
    x, r = (torch.randn(700, C, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = (1 + 0.2 * torch.randn(C, generator=g, device="cuda")).to(dtype)
    _check_norm(x, w)
    _check_norm(x, w, residual=r)
    _check_norm(x, None)


@pytest.mark.parametrize("D,Hkv,G", [(128, 2, 4), (64, 1, 5)])
def test_attend_prompts(D, Hkv, G):
    """Prompts of hundreds of tokens, on an empty and on a held cache."""
    from test_gpu_kvcache import _check_attend

    _check_attend(2, 515, Hkv, G, D, 64, [0, 700], [515, 300], seed=D, stale=0x7F)
