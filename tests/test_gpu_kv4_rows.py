"""Attention of many rows over the 4-bit cache: what a launch takes from earlier ones, small
weights, and the form for 33 to 128 rows a kv head, whose two streams take every other tile of
keys.  That form serves block tables of many tiles; here tables of 4 million tokens, of which the
sequences use the first few columns, send calls of any length to it.

Tolerances as in test_gpu_kv4.py."""

import ctypes
import math

import pytest
import torch

from _e4m3_ref import E4M3, attention, check_close
from _fp4_ref import values_of
from test_gpu_kv4 import _bound, _cache, _check_attend, _gen, _i32, _table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _setup():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    import voyager_b200  # noqa: F401

    yield


def _raw_attend(q, cache, bt, held, fill):
    """One call of the C entry with a workspace that holds `fill` in every word and no counters."""
    from voyager_b200 import _lib

    lib = _lib.load()
    B, T, H, D = q.shape
    Hkv, page, width = cache.k_codes.shape[1], cache.k_codes.shape[2], bt.shape[1]
    floats, counters = ctypes.c_int64(), ctypes.c_int64()
    assert lib.vq_attn_kv4_workspace(B, T, H, Hkv, D, page, width, ctypes.byref(floats), ctypes.byref(counters)) == 0
    assert counters.value == 0  # many rows: this kernel's counters are its workspace's
    work = torch.full((floats.value,), fill, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, math.nan)
    st = lib.vq_attn_kv4(q.data_ptr(), (ctypes.c_int64 * 3)(*q.stride()[:3]), B, T, H, Hkv, D, cache.k_codes.data_ptr(),
                         cache.v_codes.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
                         cache.k_factor.data_ptr(), cache.v_factor.data_ptr(), cache.k_codes.shape[0], page,
                         bt.data_ptr(), width, held.data_ptr(), None, 1 / math.sqrt(D), work.data_ptr(), floats.value,
                         None, 0, out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert st == 0, _lib.STATUS.get(st, st)
    return out


# heads taken whole off a counter; heads cut and joined; two streams of one row tile, cut and joined
@pytest.mark.parametrize("B,T,Hkv,G,D,held", [(40, 60, 8, 4, 64, 300), (2, 200, 2, 4, 128, 3000), (40, 30, 8, 4, 128, 700)])
def test_attend4_many_rows_start_from_any_workspace(B, T, Hkv, G, D, held):
    """Whatever an earlier launch left, one whose waits gave up included: no head is skipped and no
    join begins early."""
    from voyager_b200 import kvcache

    bt = _table(B, -(-(held + T) // 64), 1)
    cache = _cache(int(bt.max()) + 1, Hkv, 64, D, 2)
    lengths = _i32([held - b for b in range(B)])
    q = torch.randn(B, T, Hkv * G, D, generator=_gen(3), device="cuda").bfloat16()
    want = kvcache.attend(q, cache, bt, lengths)
    assert not bool(want.isnan().any())
    for fill in (0, 1, 7, 0x7F7F7F7F, -1):
        assert torch.equal(_raw_attend(q, cache, bt, lengths, fill), want)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G,B", [(1, 4, 1), (200, 2, 1), (30, 4, 40)])
@pytest.mark.parametrize("less", [33, 36])
def test_attend4_small_weights_on_large_values(T, G, B, D, less):
    """Small weights on large values, where the large weight's values are 0.  The first key's score
    is `less` above all others' in base 2; its weight is 1, the others' 2^-less each, and only they
    have values.  The largest weight is at least 2^11 in f16 (2^15 with up to 16 rows a kv head),
    whose steps are 2^-24 at the least, so a weight is off by at most 2^-25 there: 2^-36 (2^-40);
    2^-11 relative where that is more, and one bf16 rounding.  Scores are sums of D products of few
    bits, so exact."""
    from voyager_b200 import kvcache

    held, Hkv = 700, 8 if B > 1 else 1
    width = -(-(held + T) // 64)
    bt = _table(B, width, 1)
    cache = _cache(int(bt.max()) + 1, Hkv, 64, D, 2, ones=True)
    cache.k_scale.copy_(torch.ones(()))
    cache.k_codes.fill_(0)
    cache.v_scale.copy_(torch.tensor(448.0))
    cache.v_codes.fill_(0x77)  # 6 and 6
    first = bt[:, 0].long()
    cache.k_codes[first, :, 0] = 0x22  # 1 and 1, the others 0
    cache.v_codes[first, :, 0] = 0
    # q . k = less / log2(e) in the first key: D columns of less / 32, scale to match
    q = torch.full((B, T, Hkv * G, D), less / 32, device="cuda").bfloat16()
    out = kvcache.attend(q, cache, bt, _i32([held] * B), scale=32 / D * math.log(2.0)).double()
    n = held + torch.arange(T, device="cuda").double()  # keys with values that a token sees
    w = 2.0 ** -less
    want = n * w * 2688.0 / (1 + n * w)
    # sm_scale * log2(e) and its product with the score round three times: less * 3 * 2^-24 in the exponent
    floor = 2.0 ** (-40 if T * G <= 16 else -36)
    err = n * 2688.0 * (floor + w * (2.0 ** -11 + less * 3 * 2.0 ** -24)) + want * 2.0 ** -8
    assert bool(((out - want[None, :, None, None]).abs() <= err[None, :, None, None]).all()), (out.max(), out.min(), want[:3])


# ---------------------------------------------------------------------------
# 33 to 128 rows a kv head, many tiles
def _wide(bt, page):
    """The same table with columns up to 4 million tokens that no sequence uses."""
    return torch.nn.functional.pad(bt, (0, (1 << 22) // page - bt.shape[1]), value=-1).contiguous()


def _many(B, T, Hkv, G, D, page, width):
    """Whether the call is the many-row kernel's, which needs no counters of the caller."""
    from voyager_b200 import _lib

    n = ctypes.c_int64(), ctypes.c_int64()
    assert _lib.load().vq_attn_kv4_workspace(B, T, Hkv * G, Hkv, D, page, width, *map(ctypes.byref, n)) == 0
    return n[1].value == 0


def _check_rows(B, T, Hkv, G, D, page, held, counts=None, seed=0, **kw):
    assert 32 < T * G <= 128
    bt = _wide(_table(B, -(-max(h + T for h in held) // page), seed + 1), page)
    assert _many(B, T, Hkv, G, D, page, bt.shape[1])
    return _check_attend(B, T, Hkv, G, D, page, held, counts, seed, bt=bt, **kw)


ROWS = [(33, 1), (5, 7), (16, 4), (13, 5), (97, 1), (4, 32), (1, 128)]


@pytest.mark.parametrize("D,page", [(128, 64), (64, 32), (128, 128), (64, 64), (128, 32)])
@pytest.mark.parametrize("T,G", ROWS)
def test_rows_lengths(T, G, D, page):
    """Heads of 1 to 7 tiles next to longer ones, ends on and beside tiles' and halves' borders, one
    stream without a tile."""
    _check_rows(4, T, 1, G, D, page, [0, 1, 63, 64], seed=T)
    _check_rows(6, T, 2, G, D, page, [max(0, n - T) for n in (127, 128, 129, 192, 256, 257)], seed=T + 1)
    _check_rows(7, T, 2, G, D, page, [max(0, 128 * n - T - 5) for n in (5, 1, 7, 3, 20, 1, 6)], seed=T + 2)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", ROWS)
def test_rows_counts(T, G, D):
    """Unequal counts, tokens without a query, sequences without a token."""
    _check_rows(6, T, 2, G, D, 32, [0, 30, 64, 700, 5, 300], [T, (T + 1) // 2, T - 1, 1, 0, T], seed=T)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(10, 4), (128, 1)])
def test_rows_long(T, G, D):
    """One head over all SMs, and several heads cut anywhere: pieces of odd and even tiles, joins."""
    _check_rows(1, T, 1, G, D, 128, [70001], seed=T)
    _check_rows(2, T, 2, G, D, 64, [20011, 9000], seed=T + 1)
    _check_rows(9, T, 3, G, D, 64, [3000 - 331 * b for b in range(9)], seed=T + 2)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hkv", [(40, 8), (150, 2)])
def test_rows_many_heads(B, Hkv, D):
    """More heads than CTAs, more sequences than a CTA keeps plans of, some empty."""
    T, G = 12, 4
    held = [(i * 7919) % 600 if i % 5 else 0 for i in range(B)]
    counts = [0 if i % 7 == 3 else T - (i * 29) % T for i in range(B)]
    _check_rows(B, T, Hkv, G, D, 64, held, counts, seed=B)
    _check_rows(B, T, Hkv, G, D, 64, [200] * B, seed=B + 1)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(10, 4), (60, 2)])
def test_rows_references_move_apart(T, G, D):
    """Keys that grow along the sequence, keys that grow in one stream's tiles only, and scores that
    jump by more than 2^8 within half a tile: the streams' references move, and apart."""
    def grow(shape):
        def edit(cache, bt):
            raw = cache.k_scale.view(torch.uint8)
            pos = torch.arange(32 * 82, device="cuda").view(82, 32)
            for p in range(int((bt[0] >= 0).sum())):
                raw[int(bt[0, p])] = shape(pos[p])[None, :, None].byte()
            cache.k_factor.fill_(0.2)
        return edit

    _check_rows(1, T, 2, G, D, 32, [2500], seed=11, edit=grow(lambda p: 0x10 + p * 0x30 // 2624), stale=False)
    for odd in (0, 1):
        _check_rows(1, T, 2, G, D, 32, [2500], seed=12, stale=False,
                    edit=grow(lambda p: 0x10 + (p // 128 % 2 == odd) * (p * 0x38 // 2624)))
    _check_rows(1, T, 2, G, D, 32, [2500], seed=13, edit=grow(lambda p: 0x20 + p * 37 % 64 // 8 * 6), stale=False,
                sharp=4.0)


@pytest.mark.parametrize("T,G", [(10, 4), (60, 2)])
def test_rows_sharp_and_scaled(T, G):
    """Large scores, flat ones, negative scale, strides."""
    _check_rows(2, T, 2, G, 128, 64, [900, 77], seed=2, sharp=8.0)
    _check_rows(2, T, 2, G, 128, 64, [900, 77], seed=3, sharp=1e-6)
    _check_rows(2, T, 2, G, 64, 64, [900, 77], seed=4, scale=-0.05, strided=True)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(10, 4), (60, 2)])
def test_rows_scales_and_factors_of_any_size(T, G, D):
    def far(cache, bt):
        for s in (cache.k_scale, cache.v_scale):
            raw = s.view(torch.uint8)
            raw.copy_(torch.where(raw == 0x7F, raw, torch.randint(1, 0x7F, raw.shape, generator=_gen(9), device="cuda").byte()))
        cache.k_factor.copy_(torch.tensor([1e-3, 3e-4]))
        cache.v_factor.copy_(torch.tensor([1e-20, 1e20]))

    _check_rows(3, T, 2, G, D, 32, [500, 1000, 64], seed=5, edit=far)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,G", [(10, 4), (60, 2)])
@pytest.mark.parametrize("held", [61, 300, 9001])
def test_rows_nan_values(D, T, G, held):
    """A NaN in K or V reaches the rows that see it and no other, in either stream's tiles, in the
    first and in the last of them, in a head that is cut."""
    def nan_at(pos, what, head):
        def edit(cache, bt):
            getattr(cache, what + "_scale").view(torch.uint8)[int(bt[0, pos // 32]), head, pos % 32, 1] = 0x7F
        return edit

    for what in "kv":
        for pos in (held + 2, held + T - 1):
            out = _check_rows(1, T, 2, G, D, 32, [held], seed=6, edit=nan_at(pos, what, 1))
            seen = pos - held
            assert not bool(out[0, :seen].isnan().any()) and bool(out[0, seen:, G:].isnan().flatten(1).any(1).all())
            assert not bool(out[0, :, :G].isnan().any())
        for pos in (5, min(200, held - 1)):
            out = _check_rows(2, T, 2, G, D, 32, [held, 40], seed=7, edit=nan_at(pos, what, 0))
            assert bool(out[0, :, :G].isnan().flatten(1).any(1).all()) and not bool(out[1].isnan().any())


@pytest.mark.parametrize("T,G", [(10, 4), (60, 2)])
def test_rows_queries_that_are_no_numbers(T, G):
    """A NaN or an infinity in a query stays in its row."""
    from voyager_b200 import kvcache

    bt, cache = _wide(_table(1, 16, 1), 64), _cache(20, 2, 64, 128, 2)
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


@pytest.mark.parametrize("T,G", [(10, 4), (60, 2)])
@pytest.mark.parametrize("D,page", [(128, 64), (64, 32)])
@pytest.mark.parametrize("width", [12, 130])
def test_rows_leave_out_pages_outside_the_cache(T, G, D, page, width):
    """The keys of a page outside the cache are not seen, whichever stream's tile it lies in; the
    plan is reported."""
    import voyager_b200
    from voyager_b200 import _lib, kvcache

    Hkv, held = 2, (width - 2) * page + 3 - T
    bt = _table(1, width, 3)
    cache = _cache(width + 2, Hkv, page, D, 4)
    for gone, bad in (((1, 4), -1), ((0, 1, 2, 3), width + 2), ((width - 2, 5), 2 ** 30)):
        bt2 = bt.clone()
        for p in gone:
            bt2[0, p] = bad
        q = torch.randn(1, T, Hkv * G, D, generator=_gen(T), device="cuda").bfloat16()
        out = kvcache.attend(q, cache, _wide(bt2, page), _i32([held]))
        with pytest.raises(_lib.VqError, match="plan"):
            voyager_b200.check_errors()
        n = held + T
        keep = torch.ones(n, dtype=torch.bool, device="cuda")
        for p in gone:
            keep[p * page:(p + 1) * page] = False
        ids = bt[0, :-(-n // page)].long()
        for h in range(Hkv):
            k, v = (values_of(x[ids, h], s.view(torch.uint8)[ids, h].view(E4M3), f[h].double()).reshape(-1, D)[:n]
                    for x, s, f in ((cache.k_codes, cache.k_scale, cache.k_factor),
                                    (cache.v_codes, cache.v_scale, cache.v_factor)))
            for t in range(T):  # a token's keys: those up to its own that are kept
                own = keep[:held + t + 1]
                kt, vt = k[:held + t + 1][own], v[:held + t + 1][own]
                want, mag = attention(q[0, t:t + 1, h * G:(h + 1) * G].double(), kt, vt, len(kt) - 1, 1 / math.sqrt(D))
                check_close(out[0, t:t + 1, h * G:(h + 1) * G], want, _bound(want, mag, vt, T * G))


@pytest.mark.parametrize("T,wide", [(10, True), (30, True), (130, False)])
def test_rows_offsets_past_32_bits(T, wide):
    """Pages beyond 2^31 bytes of the cache, read by either form of the many-row kernel."""
    from voyager_b200 import kvcache

    pages, Hkv, page, D = 36000, 4, 128, 128
    cache = kvcache.KVCache4.empty(pages, Hkv, D, page)
    bt = _i32([[pages - 1, 17, pages - 3], [pages - 2, pages - 4, 3]])
    g = _gen(8)
    for t in (cache.k_codes, cache.v_codes):
        for p in bt.flatten().tolist():
            t[p] = torch.randint(0, 256, t[p].shape, generator=g, device="cuda").byte()
    if wide:
        bt = _wide(bt, page)
    assert _many(2, T, Hkv, 4, D, page, bt.shape[1])
    _check_attend(2, T, Hkv, 4, D, page, [300 - T, 383 - T], cache=cache, bt=bt, seed=9)


@pytest.mark.parametrize("T,G,D", [(10, 4, 128), (60, 2, 64)])
def test_rows_streams_and_graphs(T, G, D):
    """Calls on two streams and in two graphs at once, heads cut; replays after the plan has changed."""
    from voyager_b200 import kvcache

    bt = _wide(_table(2, 160, 1), 64)
    cache = _cache(330, 2, 64, D, 2)
    qs = [torch.randn(2, T, 2 * G, D, generator=_gen(i), device="cuda").bfloat16() for i in range(2)]
    held = _i32([9000, 3000])
    want = [kvcache.attend(q, cache, bt, held) for q in qs]
    short = [kvcache.attend(q, cache, bt, held - 2500) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
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
    for less, expect in ((0, want), (2500, short), (0, want)):
        held.copy_(_i32([9000 - less, 3000 - less]))
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, expect))


def test_rows_empty_plans():
    """No new token anywhere, no key but the token's own, and lengths that do not fit."""
    import voyager_b200
    from voyager_b200 import _lib, kvcache

    _check_rows(3, 10, 2, 4, 64, 32, [0, 0, 50], [0, 0, 0])
    _check_rows(3, 40, 2, 1, 128, 32, [0, 0, 0], [1, 0, 40])
    bt, cache = _wide(_table(1, 4, 1), 32), _cache(8, 2, 32, 64, 2)
    q = torch.randn(1, 10, 8, 64, generator=_gen(1), device="cuda").bfloat16()
    for held, count in ((-1, 10), (5, -2), (5, 11), (1 << 22, 10)):
        out = kvcache.attend(q, cache, bt, _i32([held]), _i32([count]))
        with pytest.raises(_lib.VqError, match="plan"):
            voyager_b200.check_errors()
        assert count == 11 or not bool(out.any())  # 11 of 10 tokens: all 10


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [4, 8])
def test_prompts_captured_and_replayed(bits):
    """Append and attention of prompts in a graph, whose kernels start under one another: replays with
    other inputs and another plan write what eager calls write."""
    from voyager_b200 import kvcache

    B, T, Hkv, G, D, page = 3, 700, 8, 4, 128, 64
    kind = kvcache.KVCache4 if bits == 4 else kvcache.KVCache
    table, bt = kvcache.rotary_table(1024, D), _table(B, 16, 1)
    w = (1 + 0.3 * torch.randn(D, generator=_gen(2), device="cuda")).bfloat16()
    xs = [torch.randn(B, T, (G + 2) * Hkv, D, generator=_gen(i), device="cuda").bfloat16() for i in range(3)]
    plans = [([0, 0, 0], [T, T, T]), ([5, 300, 64], [T, 1, 650]), ([0, 63, 0], [0, T, 33])]
    x, held, new = xs[0].clone(), _i32(plans[0][0]), _i32(plans[0][1])

    def step(cache):
        q, k, v = x.split([G * Hkv, Hkv, Hkv], 2)
        q = kvcache.rope_append(q, k, v, table, cache, bt, held, new, q_norm=w, k_norm=w)
        return kvcache.attend(q, cache, bt, held, new)

    eager, own = (kind.empty(B * 16 + 2, Hkv, D, page) for _ in range(2))
    step(kind.empty(B * 16 + 2, Hkv, D, page))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(own)
    for data, (h, n) in zip(xs, plans):
        x.copy_(data), held.copy_(_i32(h)), new.copy_(_i32(n))
        want = step(eager)
        graph.replay()
        assert torch.equal(out, want)
        for n in ("k_codes", "v_codes", "k_scale", "v_scale"):
            assert torch.equal(getattr(own, n).view(torch.uint8), getattr(eager, n).view(torch.uint8))
