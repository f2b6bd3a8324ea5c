"""Host side of the 4-bit cache's operators and of the head norms, without a
GPU: refusals of the entry points and of the C ABI before any launch, and the
references that the GPU tests compare with."""

import ctypes
import math

import pytest
import torch

from _fp4_ref import E2M1, codes_of, e2m1, values_of
from voyager_b200 import _lib, kvcache

P = 0x1000  # never dereferenced: the calls are refused or do nothing


def test_reference_rounding():
    """Each value to the nearest code; every tie to the even one."""
    for i, (a, b) in enumerate(zip(E2M1, E2M1[1:])):
        mid = (a + b) / 2
        x = torch.tensor([a, mid - 1e-9, mid, mid + 1e-9, b, 7.0, math.inf], dtype=torch.float64)
        want = torch.tensor([a, a, a if i % 2 == 0 else b, b, b, 6.0, 6.0], dtype=torch.float64)
        assert torch.equal(e2m1(x), want) and torch.equal(e2m1(-x), -want)
    raw = torch.arange(256, dtype=torch.uint8)
    v = codes_of(raw).view(256, 2)
    assert v[0x71].tolist() == [0.5, 6.0] and v[0xA9].tolist() == [-0.5, -1.0]
    s = torch.full((1, 1), 0.5).to(torch.float8_e4m3fn)
    assert values_of(raw[:8][None], s, 4.0).tolist() == [[2 * x for x in v[:8].flatten().tolist()]]


def test_cpu_tensors_are_refused():
    cache = kvcache.KVCache4.empty(1, 1, 64, 32, device="cpu")
    q = torch.zeros(1, 1, 1, 64).bfloat16()
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        kvcache.attend(q, cache, i[None], i)
    with pytest.raises(NotImplementedError):
        kvcache.rope_append(q, q, q, kvcache.rotary_table(32, 64, device="cpu"), cache, i[None], i)
    with pytest.raises(NotImplementedError):
        kvcache.unpack(cache)
    with pytest.raises(ValueError):
        kvcache.KVCache4.empty(1, 1, 64, 16, device="cpu")
    with pytest.raises(AttributeError):
        kvcache.unpack(None)


def _rope(lib, fn="vq_rope_append_kv4", **kw):
    a = dict(q=P, k=P, v=P, strides=(ctypes.c_int64 * 9)(*[128] * 9), dtype=_lib.VQ_BF16, table=P, positions=64,
             rot=128, il=0, batch=1, tokens=0, heads=4, kv=2, D=128, bt=P, width=1, lengths=P, counts=None, pages=1,
             page=64, qn=None, kn=None, eps=1e-6, q_out=P, kc=P, vc=P, ks=P, vs=P, kf=P, vf=P)
    if fn.endswith("norm"):
        del a["kf"], a["vf"]
    a.update(kw)
    return getattr(lib, fn)(*a.values(), None)


@pytest.mark.parametrize("fn", ["vq_rope_append_kv4", "vq_rope_append_kv8_norm"])
def test_rope_abi(fn):
    lib = _lib.load()

    def go(**kw):
        return _rope(lib, fn, **kw)

    assert go() == 0 and go(batch=0, tokens=1) == 0
    assert go(dtype=_lib.VQ_F16) == 2 and go(D=96) == 2 and go(page=16) == 2
    for kw in ({"batch": -1}, {"heads": 3}, {"heads": 0}, {"kv": 0}, {"rot": 0}, {"rot": 24}, {"rot": 144},
               {"pages": 1 << 40}, {"width": -1}):
        assert go(**kw) == 1, kw
    for n in ("q", "k", "v", "table", "bt", "lengths", "q_out", "kc", "vc", "ks", "vs"):
        assert go(tokens=1, **{n: None}) == 6, n
    assert go(tokens=1, positions=63) == 5
    for n in ("q", "kc", "qn", "kn", "table"):
        assert go(tokens=1, **{n: P + 8}) == 3, n
    assert go(tokens=1, q_out=P + 16) == 3
    assert go(tokens=1, strides=(ctypes.c_int64 * 9)(*[129] * 9)) == 3


def test_rope_abi_of_four_bits():
    lib = _lib.load()
    assert _rope(lib, tokens=1, kf=None) == 6 and _rope(lib, tokens=1, vf=None) == 6
    assert _rope(lib, tokens=1 << 20, batch=1 << 12) == 1  # tokens past 31 bits


def test_unpack_abi():
    lib = _lib.load()
    assert lib.vq_kv4_unpack(None, None, 0, None, None, None) == 0
    assert lib.vq_kv4_unpack(P, P, -16, P, P, None) == 1 and lib.vq_kv4_unpack(P, P, 8, P, P, None) == 1
    for i in range(4):
        a = [P] * 4
        a[i] = None
        assert lib.vq_kv4_unpack(a[0], a[1], 16, a[2], a[3], None) == 6
        for off in (4, 16) if i > 1 else (4,):  # whole sectors are written
            a[i] = P + off
            assert lib.vq_kv4_unpack(a[0], a[1], 16, a[2], a[3], None) == 3


def test_attend_abi():
    lib = _lib.load()
    f, c = ctypes.c_int64(), ctypes.c_int64()
    B = ctypes.byref

    def size(b=2, t=1, h=32, kv=8, D=128, page=64, width=2000):
        st = lib.vq_attn_kv4_workspace(b, t, h, kv, D, page, width, B(f), B(c))
        return st, f.value, c.value

    st, floats, counters = size()
    assert st == 0 and counters >= 16 and floats > 0
    assert size(width=1)[1] <= floats
    assert size(h=31)[0] == 1 and size(kv=0)[0] == 1 and size(b=-1)[0] == 1
    assert lib.vq_attn_kv4_workspace(1, 1, 1, 1, 64, 64, 1, None, B(c)) == 6

    def go(**kw):
        a = dict(q=P, strides=(ctypes.c_int64 * 3)(128, 128, 128), batch=1, tokens=0, heads=4, kv=2, D=128, kc=P, vc=P,
                 ks=P, vs=P, kf=P, vf=P, pages=1, page=64, bt=P, width=1, lengths=P, counts=None, scale=1.0, ws=None,
                 wsn=0, done=P, donen=2, out=P)
        a.update(kw)
        return lib.vq_attn_kv4(*a.values(), None)

    assert go() == 0 and go(batch=0, tokens=3) == 0
    assert go(D=96) == 2 and go(page=16) == 2
    assert go(heads=5) == 1 and go(batch=1 << 25) == 1 and go(pages=1 << 40) == 1 and go(tokens=-1) == 1
    for T in (1, 40):
        for n in ("q", "strides", "kc", "vc", "ks", "vs", "kf", "vf", "bt", "lengths", "done", "out"):
            assert go(tokens=T, donen=100, **{n: None}) == 6, n
        for n in ("q", "kc", "vc", "ks", "vs", "out"):
            assert go(tokens=T, donen=100, **{n: P + 8}) == 3, n
        assert go(tokens=T, strides=(ctypes.c_int64 * 3)(4, 128, 128)) == 3
        assert go(tokens=T, donen=1) == 1                    # too few counters
        assert go(tokens=T, donen=100) == 1                  # no workspace
