"""Attention of many rows over the 4-bit cache: what a launch takes from earlier ones, and small
weights.

Tolerances as in test_gpu_kv4.py."""

import ctypes
import math

import pytest
import torch

from test_gpu_kv4 import _cache, _gen, _i32, _table

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
