"""Host side of the cached-decoding operators, without a GPU: the rotary
tables against their formulas, and the C ABI's refusals before any launch."""

import ctypes
import math

import pytest
import torch

from voyager_b200 import _lib, fp8block, kvcache

P = 0x1000  # never dereferenced: the calls are refused or do nothing


def test_rotary_table_plain_and_linear():
    for rot, theta in ((64, 10000.0), (128, 500000.0)):
        t = kvcache.rotary_table(50, rot, theta, device="cpu")
        assert t.shape == (50, rot // 2, 2) and t.dtype == torch.float32
        for p in (0, 1, 49):
            for i in (0, 3, rot // 2 - 1):
                a = p * theta ** (-2 * i / rot)
                assert t[p, i, 0] == pytest.approx(math.cos(a), abs=1e-7)
                assert t[p, i, 1] == pytest.approx(math.sin(a), abs=1e-7)
        lin = kvcache.rotary_table(100, rot, theta, scaling="linear", factor=2.0, device="cpu")
        assert torch.equal(lin[::2], t)


def test_rotary_table_long_contexts():
    rot, n, f = 128, 4096, 8.0
    freq = [10000.0 ** (-2 * i / rot) for i in range(rot // 2)]

    def angles(**kw):
        t = kvcache.rotary_table(2, rot, factor=f, device="cpu", **kw).double()
        return torch.atan2(t[1, :, 1], t[1, :, 0]), t[1].norm(dim=-1)

    a, amp = angles(scaling="ntk")
    assert a[0] == pytest.approx(1.0, rel=1e-6) and a[-1] == pytest.approx(freq[-1] / f, rel=1e-5)
    assert amp.sub(1).abs().max() < 1e-6
    a, amp = angles(scaling="smooth", original=n, low=1.0, high=4.0)
    for i, w in enumerate(freq):
        turns = n * w / (2 * math.pi)
        k = min(max((turns - 1) / 3, 0), 1)
        assert a[i] == pytest.approx(w * k + w / f * (1 - k), rel=1e-5)
    a, amp = angles(scaling="parts", original=n, low=1.0, high=32.0)
    assert amp.sub(0.1 * math.log(f) + 1).abs().max() < 1e-6
    for i, w in enumerate(freq):
        turns = n * w / (2 * math.pi)
        if turns > 40:
            assert a[i] == pytest.approx(w, rel=1e-6)
        if turns < 0.9:
            assert a[i] == pytest.approx(w / f, rel=1e-5)
    assert all(a[i] >= a[i + 1] for i in range(rot // 2 - 1))


@pytest.mark.parametrize("args,kw", [((8, 3), {}), ((8, 0), {}), ((-1, 4), {}), ((8, 4), {"scaling": "other"}),
                                     ((8, 4), {"scaling": "linear", "factor": 0.5}),
                                     ((8, 4), {"scaling": "parts", "factor": 2.0}),
                                     ((8, 4), {"scaling": "smooth", "factor": 2.0, "original": 9, "low": 4.0, "high": 2.0})])
def test_rotary_table_refusals(args, kw):
    with pytest.raises(ValueError):
        kvcache.rotary_table(*args, device="cpu", **kw)


def test_cpu_tensors_are_refused():
    x = torch.randn(2, 128)
    with pytest.raises(NotImplementedError):
        fp8block.rmsnorm_quantize(x, torch.ones(128))
    with pytest.raises(NotImplementedError):
        fp8block.quantize(x)
    c, s = x.to(torch.float8_e4m3fn), torch.ones(2, 1)
    with pytest.raises(NotImplementedError):
        fp8block.linear(c, s, c, torch.ones(1, 1))
    cache = kvcache.KVCache.empty(1, 1, 64, 32, device="cpu")
    q = torch.zeros(1, 1, 1, 64).bfloat16()
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        kvcache.attend(q, cache, i[None], i)
    with pytest.raises(NotImplementedError):
        kvcache.rope_append(q, q, q, kvcache.rotary_table(32, 64, device="cpu"), cache, i[None], i)


def test_quantize_weight_on_the_host():
    w = torch.randn(130, 200, generator=torch.Generator().manual_seed(0))
    w[128:] = 0
    codes, scale = fp8block.quantize_weight(w)
    assert scale.shape == (2, 2) and bool((scale[1] == 1).all()) and not bool(codes[128:].float().any())
    assert scale[0, 0] == w[:128, :128].abs().max() / 448
    with pytest.raises(ValueError):
        fp8block.quantize_weight(w[0])


def _norm(lib, **kw):
    a = dict(x=P, ldx=256, r=None, ldr=0, w=P, dtype=_lib.VQ_BF16, rows=0, cols=256, eps=1e-5, codes=P, scale=P,
             hidden=None)
    a.update(kw)
    return lib.vq_norm_quantize_fp8(*a.values(), None)


def test_norm_abi():
    lib = _lib.load()
    assert _norm(lib) == 0  # no rows: nothing to do
    assert _norm(lib, rows=-1) == 1 and _norm(lib, cols=0) == 1 and _norm(lib, rows=1 << 31) == 1
    assert _norm(lib, dtype=_lib.VQ_F16) == 2
    assert _norm(lib, rows=1, x=None) == 6 and _norm(lib, rows=1, codes=None) == 6
    assert _norm(lib, rows=1, r=P, ldr=256) == 6  # a residual without hidden
    assert _norm(lib, rows=1, ldx=255) == 5 and _norm(lib, rows=1, r=P, ldr=8, hidden=P) == 5
    assert _norm(lib, rows=1, x=P + 1) == 3 and _norm(lib, rows=1, scale=P + 2) == 3


def test_linear_abi():
    lib = _lib.load()

    def go(x=P, sx=P, w=P, sw=P, bias=None, M=0, N=128, K=128, out=P, ldo=128):
        return lib.vq_linear_fp8_block(x, sx, w, sw, bias, M, N, K, out, ldo, None)

    assert go() == 0
    assert go(M=-1) == 1 and go(N=0) == 1 and go(K=0) == 1 and go(M=1 << 30) == 1
    assert go(K=24) == 2
    assert go(M=1, ldo=64) == 5
    for n in ("x", "sx", "w", "sw", "out"):
        assert go(M=1, **{n: None}) == 6
    assert go(M=1, x=P + 8) == 3 and go(M=1, w=P + 1) == 3 and go(M=1, sx=P + 2) == 3 and go(M=1, out=P + 1) == 3


def _rope(lib, **kw):
    a = dict(q=P, k=P, v=P, strides=(ctypes.c_int64 * 9)(*[128] * 9), dtype=_lib.VQ_BF16, table=P, positions=64,
             rot=128, il=0, batch=1, tokens=0, heads=4, kv=2, D=128, bt=P, width=1, lengths=P, counts=None, pages=1,
             page=64, q_out=P, kc=P, vc=P, ks=P, vs=P)
    a.update(kw)
    return lib.vq_rope_append_kv8(*a.values(), None)


def test_rope_abi():
    lib = _lib.load()
    assert _rope(lib) == 0 and _rope(lib, batch=0, tokens=1) == 0
    assert _rope(lib, dtype=_lib.VQ_F16) == 2 and _rope(lib, D=96) == 2 and _rope(lib, page=16) == 2
    for kw in ({"batch": -1}, {"heads": 3}, {"heads": 0}, {"kv": 0}, {"rot": 0}, {"rot": 24}, {"rot": 144},
               {"pages": 1 << 40}, {"width": -1}):
        assert _rope(lib, **kw) == 1, kw
    for n in ("q", "k", "v", "table", "bt", "lengths", "q_out", "kc", "vc", "ks", "vs"):
        assert _rope(lib, tokens=1, **{n: None}) == 6, n
    assert _rope(lib, tokens=1, batch=1 << 20, heads=32, kv=32) == 1  # 2^26 blocks, up to 32 threads each
    assert _rope(lib, tokens=1, positions=63) == 5
    assert _rope(lib, tokens=1, q=P + 8) == 3
    assert _rope(lib, tokens=1, strides=(ctypes.c_int64 * 9)(*[129] * 9)) == 3


def test_attend_abi():
    lib = _lib.load()
    f, c = ctypes.c_int64(), ctypes.c_int64()
    B = ctypes.byref

    def size(b=2, t=1, h=32, kv=8, D=128, page=64, width=2000):
        st = lib.vq_attn_kv8_workspace(b, t, h, kv, D, page, width, B(f), B(c))
        return st, f.value, c.value

    st, floats, counters = size()
    assert st == 0 and counters >= 16 and floats > 0
    assert size(width=1)[1] <= floats
    assert size(t=12, h=64)[2] >= 16 * 6
    assert size(h=31)[0] == 1 and size(kv=0)[0] == 1 and size(b=-1)[0] == 1
    assert lib.vq_attn_kv8_workspace(1, 1, 1, 1, 64, 64, 1, None, B(c)) == 6

    def go(**kw):
        a = dict(q=P, strides=(ctypes.c_int64 * 3)(128, 128, 128), batch=1, tokens=0, heads=4, kv=2, D=128, kc=P, vc=P,
                 ks=P, vs=P, pages=1, page=64, bt=P, width=1, lengths=P, counts=None, scale=1.0, ws=None, wsn=0,
                 done=P, donen=2, out=P)
        a.update(kw)
        return lib.vq_attn_kv8(*a.values(), None)

    assert go() == 0 and go(batch=0, tokens=3) == 0
    assert go(D=96) == 2 and go(page=16) == 2
    assert go(heads=5) == 1 and go(batch=1 << 25) == 1 and go(pages=1 << 40) == 1 and go(tokens=-1) == 1
    for n in ("q", "strides", "kc", "vc", "ks", "vs", "bt", "lengths", "done", "out"):
        assert go(tokens=1, **{n: None}) == 6, n
    assert go(tokens=1, q=P + 8) == 3 and go(tokens=1, strides=(ctypes.c_int64 * 3)(4, 128, 128)) == 3
    assert go(tokens=1, donen=1) == 1                    # too few counters
    assert go(tokens=1, donen=2) == 1                    # no workspace
