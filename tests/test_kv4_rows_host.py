"""Attention of many rows over the 4-bit cache without a GPU: which kernel a call takes, and the
refusals of the many-row one."""

import ctypes

import pytest

from voyager_b200 import _lib

P = 0x1000  # never dereferenced: the calls are refused


def _sizes(batch, tokens, group, kv, dim, width, page=64):
    f, c = ctypes.c_int64(), ctypes.c_int64()
    assert _lib.load().vq_attn_kv4_workspace(batch, tokens, kv * group, kv, dim, page, width, ctypes.byref(f),
                                             ctypes.byref(c)) == 0
    return f.value, c.value


# head_dim, rows, sequences (8 kv heads), tokens of the table, then us of the few-row and the many-row
# kernel with every sequence as long as the table, and with lengths spread evenly below that
MEASURED = [
    (128, 48, 16, 2048, (54, 44), (33, 36)), (128, 48, 4, 16064, (80, 61), (40, 44)),
    (128, 48, 64, 1024, (107, 84), (57, 86)), (128, 128, 4, 1024, (30, 31), (20, 29)),
    (128, 128, 4, 4032, (61, 40), (32, 37)), (128, 128, 64, 1024, (259, 90), (98, 82)),
    (64, 48, 4, 16064, (54, 50), (32, 37)), (64, 48, 64, 1024, (69, 66), (42, 65)),
    (64, 128, 4, 4032, (45, 30), (25, 27)), (64, 128, 64, 1024, (187, 69), (72, 60)),
    (64, 80, 64, 256, (54, 34), (34, 34)), (128, 80, 64, 256, (75, 46), (47, 45)),
]


@pytest.mark.parametrize("dim,rows,batch,tokens,equal,unequal", MEASURED)
def test_choice_follows_the_measurements(dim, rows, batch, tokens, equal, unequal):
    """The kernel taken is at most a third slower than the other one at these points (times rounded to
    1 us), be the lengths equal or not, which the host does not know."""
    many = _sizes(batch, rows // 8, 8, 8, dim, tokens // 64)[1] == 0
    for here, there in (equal, unequal):
        taken, left = (there, here) if many else (here, there)
        assert (taken - 0.5) / (left + 0.5) <= 4 / 3


def test_choice_at_its_ends():
    for dim in (64, 128):
        for width in (1, 40, 60000):
            assert _sizes(8, 4, 8, 8, dim, width)[1] > 0      # 32 rows
            assert _sizes(8, 129, 1, 8, dim, width)[1] == 0   # 129 rows
        assert _sizes(1, 128, 1, 1, dim, 1)[1] > 0 and _sizes(8, 33, 1, 8, dim, 60000)[1] == 0


def test_many_rows_abi():
    lib = _lib.load()
    floats, counters = _sizes(1, 200, 2, 2, 128, 1)
    assert counters == 0

    def go(**kw):
        a = dict(q=P, strides=(ctypes.c_int64 * 3)(128, 128, 128), batch=1, tokens=200, heads=4, kv=2, D=128, kc=P, vc=P,
                 ks=P, vs=P, kf=P, vf=P, pages=1, page=64, bt=P, width=1, lengths=P, counts=None, scale=1.0, ws=P,
                 wsn=floats - 1, done=None, donen=0, out=P)
        a.update(kw)
        return lib.vq_attn_kv4(*a.values(), None)

    for n in ("q", "strides", "kc", "vc", "ks", "vs", "kf", "vf", "bt", "lengths", "out"):
        assert go(**{n: None}) == 6, n
    for n in ("q", "kc", "vc", "ks", "vs", "ws"):
        assert go(**{n: P + 8}) == 3, n
    assert go(out=P + 16) == 3
    assert go(strides=(ctypes.c_int64 * 3)(4, 128, 128)) == 3
    assert go() == 1 and go(wsn=0) == 1 and go(ws=None, wsn=floats) == 1       # a workspace too small, none
    assert go(batch=1 << 12, width=1 << 20, wsn=1 << 40) == 1                    # tiles past 31 bits
    assert go(width=1 << 26, wsn=1 << 40) == 1                                   # a table past 31 bits
