"""The cached decoder's head norms: each layer's own weights, the queries' on the queries and the
keys' on the keys, against layers whose heads are normalised in float64 before an append without
norms.

Tolerances.  Both runs share everything up to the first append.  There a normalised and turned value
is a float32 within 19 * 2^-24 of its head's largest (test_gpu_kv4.py), by hand the rounding of a
float64, so that queries, as bfloat16, differ by one rounding step at most: 2^-7 of the value and
2^-18 of the head's largest.  A key's code differs only where its quotient lies that close to the
border between two codes: 2^-19 of the largest, whose steps are 2^-4 of it or more, for fewer than
2^-14 of the codes; sixteen that share a scale on a border too, fewer than 2^-10 in all.  After all
layers: below a bfloat16 rounding of the attention's outputs, which test_gpu_decode4.py bounds by
6 % of what the layers add."""

import pytest
import torch

from _fp4_ref import head_norm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _setup():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    import voyager_b200  # noqa: F401

    yield


@pytest.mark.parametrize("only", ["qk", "q", "k"])
@pytest.mark.parametrize("bits,kv_heads,head_dim", [(4, 2, 128), (4, 8, 64), (8, 2, 128)])
def test_head_norms_are_the_layers_own(bits, kv_heads, head_dim, only, monkeypatch):
    from voyager_b200 import kvcache
    from voyager_b200.decode import CachedDecoder
    from voyager_b200.decoder import DecoderConfig, init_weights

    cfg = DecoderConfig(layers=2, hidden=8 * head_dim, heads=8, ffn=1408)
    weights = init_weights(cfg, 3, "cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    for w in weights:
        for n in only:
            w[n + "_norm"] = (1 + 0.5 * torch.randn(head_dim, generator=g, device="cuda")).bfloat16()
    dec = CachedDecoder(cfg, weights, kv_heads=kv_heads, max_positions=256, cache_bits=bits)
    B, T = 2, 150
    x = torch.randn(B, T, cfg.hidden, generator=g, device="cuda").bfloat16()
    bt = torch.randperm(8, generator=g, device="cuda").view(B, 4).int()
    held, counts = (torch.tensor(n, dtype=torch.int32, device="cuda") for n in ([0, 0], [T, 97]))
    append, attend, queries = kvcache.rope_append, kvcache.attend, []

    def seen(q, *args):
        queries.append(q)
        return attend(q, *args)

    layer = iter(weights)

    def by_hand(q, k, v, table, cache, block_table, lengths, counts, **_):
        w = next(layer)
        q, k = (head_norm(t.double(), w.get(n), cfg.eps).float() for t, n in ((q, "q_norm"), (k, "k_norm")))
        return append(q, k, v.float(), table, cache, block_table, lengths, counts).bfloat16()

    monkeypatch.setattr(kvcache, "attend", seen)
    own, hand = dec.caches(8), dec.caches(8)
    y = dec.step(x, own, bt, held, counts)
    monkeypatch.setattr(kvcache, "rope_append", by_hand)
    want = dec.step(x, hand, bt, held, counts)
    assert len(queries) == 4 and next(layer, None) is None
    a, b = queries[0].float(), queries[2].float()
    assert bool(((a - b).abs() <= b.abs() * 2.0 ** -7 + b.abs().amax(-1, keepdim=True) * 2.0 ** -18).all())
    for n in ("k_codes", "k_scale", "v_codes", "v_scale"):
        a, b = (getattr(c[0], n).view(torch.uint8) for c in (own, hand))
        assert float((a != b).float().mean()) < (2.0 ** -10 if n[0] == "k" else 2.0 ** -30)
    for i in range(B):
        n = int(counts[i])
        base = x[i, :n].float()
        diff = y[i, :n].float() - want[i, :n].float()
        assert float(diff.norm() / (want[i, :n].float() - base).norm()) < 0.06
