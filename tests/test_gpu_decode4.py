"""The cached decoder on a 4-bit cache, with and without normalised heads: its
operators run together, against the same layers with the attention computed in
64 bits from the values that the cache holds, token by token against the prompt
in one step, and captured.

Tolerances.  Against the 64-bit attention the two runs share every quantized
operand up to the attention's bf16 outputs, which differ by at most one rounding
(2^-8); requantized to E4M3 (a step is 2^-3 relative at most, 2^-4 off) an output
near a border moves by a step, which happens to about one in 2^-8 / 2^-3 = 1/32 of
them: sqrt(1/32) * 2^-3 = 2.2 % of the attention's part of the residual stream,
and as much again from the later layer's inputs; 6 % of what the layers add is
allowed.  Token by token the cache holds the prompt's bytes where its inputs are
equal; they differ by bf16 roundings of sums, which move a 4-bit code (a step is
at most half its value, 1/3 of a block's largest) for about 2^-8 / 2^-2 = 1/64 of
the values: sqrt(1/64) / 3 = 4 % of keys and values, and 2.2 % for the E4M3
operands; 8 % of the layers' sum is allowed."""

import math

import pytest
import torch

from _fp4_ref import values_of

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _setup():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    import voyager_b200  # noqa: F401

    yield


def _decoder(kv_heads, head_dim, norms, heads=8, layers=2):
    from voyager_b200.decode import CachedDecoder
    from voyager_b200.decoder import DecoderConfig, init_weights

    cfg = DecoderConfig(layers=layers, hidden=heads * head_dim, heads=heads, ffn=1408)
    weights = init_weights(cfg, 3, "cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    for w in weights:
        for n in ("q_norm", "k_norm") if norms else ():
            w[n] = (1 + 0.2 * torch.randn(head_dim, generator=g, device="cuda")).bfloat16()
    return cfg, CachedDecoder(cfg, weights, kv_heads=kv_heads, max_positions=640, cache_bits=4)


def _attention(q, cache, bt, held, counts, G):
    """The attention of q [B, T, H, D] over the cache in 64 bits, as bfloat16."""
    B, T, H, D = q.shape
    out = torch.zeros_like(q)
    for b in range(B):
        c, n = int(counts[b]), int(held[b] + counts[b])
        ids = bt[b, :-(-n // cache.k_codes.shape[2])].long()
        for h in range(H // G):
            k, v = (values_of(x[ids, h], s.view(torch.uint8)[ids, h].view(E4M3), f[h].double()).reshape(-1, D)[:n]
                    for x, s, f in ((cache.k_codes, cache.k_scale, cache.k_factor),
                                    (cache.v_codes, cache.v_scale, cache.v_factor)))
            s = torch.einsum("tgd,kd->tgk", q[b, :c, h * G:(h + 1) * G].double(), k) / math.sqrt(D)
            late = torch.arange(n, device="cuda") > int(held[b]) + torch.arange(c, device="cuda")[:, None]
            out[b, :c, h * G:(h + 1) * G] = (torch.softmax(s.masked_fill(late[:, None], -math.inf), -1) @ v).bfloat16()
    return out


@pytest.mark.parametrize("kv_heads,head_dim,norms", [(8, 128, False), (2, 64, True), (2, 128, True)])
def test_prompt_and_steps(kv_heads, head_dim, norms, monkeypatch):
    from voyager_b200 import kvcache

    cfg, dec = _decoder(kv_heads, head_dim, norms)
    g = torch.Generator(device="cuda").manual_seed(1)
    S, B = 150, 2
    x = torch.randn(B, S, cfg.hidden, generator=g, device="cuda").bfloat16()
    counts = torch.tensor([S, 97], dtype=torch.int32, device="cuda")
    bt = torch.randperm(20, generator=g, device="cuda")[:20].view(B, 10).int()
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    y = dec.step(x, dec.caches(20), bt, zero, counts)
    with monkeypatch.context() as m:
        m.setattr(kvcache, "attend", lambda q, c, t, held, n: _attention(q, c, t, held, n, cfg.heads // kv_heads))
        exact = dec.step(x, dec.caches(20), bt, zero, counts)
    for b in range(B):
        n = int(counts[b])
        base = x[b, :n].float()
        want = exact[b, :n].float() - base
        assert float((y[b, :n].float() - base - want).norm() / want.norm()) < 0.06
    # the last 40 tokens again, one at a time and then five at a time
    caches = dec.caches(20)
    lengths = counts - 40
    dec.step(x, caches, bt, zero, lengths)
    at, steps = lengths.clone(), []
    rows = torch.arange(B, device="cuda")[:, None]
    for T in [1] * 20 + [5] * 4:
        new = at[:, None] + torch.arange(T, device="cuda")
        steps.append(dec.step(x[rows, new], caches, bt, at))
        at += T
    new = lengths[:, None] + torch.arange(40, device="cuda")
    base = x[rows, new].float()
    want = y[rows, new].float() - base
    assert float((torch.cat(steps, 1).float() - base - want).norm() / want.norm()) < 0.08


def test_norms_change_nothing_else():
    """Head norms with the E4M3 cache: weights of one and heads whose mean square is
    one already give what no norm gives, up to roundings (as in the E4M3 decoder's
    own test: 3 %)."""
    from voyager_b200.decode import CachedDecoder
    from voyager_b200.decoder import DecoderConfig, init_weights

    cfg = DecoderConfig(layers=1, hidden=1024, heads=8, ffn=1408)
    w = init_weights(cfg, 3, "cuda")
    x = torch.randn(1, 70, 1024, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    bt = torch.arange(2, device="cuda").int().view(1, 2)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    ys = []
    for norms in (False, True):
        # scores do not depend on the queries' size where the norm undoes it
        ws = [dict(v, q_norm=torch.ones(128, device="cuda").bfloat16(), k_norm=torch.ones(128, device="cuda").bfloat16())
              if norms else dict(v) for v in w]
        for v in ws:
            if norms:
                v["q"], v["k"] = v["q"] * 3, v["k"] * 0.25
        dec = CachedDecoder(cfg, ws, kv_heads=8, max_positions=128)
        ys.append(dec.step(x, dec.caches(2), bt, zero))
    big = [dict(v, q=v["q"] * 12, k=v["k"] * 2, q_norm=torch.ones(128, device="cuda").bfloat16(),
                k_norm=torch.ones(128, device="cuda").bfloat16()) for v in w]
    dec = CachedDecoder(cfg, big, kv_heads=8, max_positions=128)
    other = dec.step(x, dec.caches(2), bt, zero)
    want = ys[1].float() - x.float()
    assert float((other.float() - ys[1].float()).norm() / want.norm()) < 0.03  # whatever the projections' size
    assert not torch.equal(ys[0], ys[1])


def test_step_in_a_graph():
    """A captured step replays with the plan advanced in place."""
    cfg, dec = _decoder(4, 64, True)
    g = torch.Generator(device="cuda").manual_seed(2)
    xs = torch.randn(6, 3, 1, cfg.hidden, generator=g, device="cuda").bfloat16()
    bt = torch.arange(30, device="cuda").view(3, 10).int()
    start = torch.tensor([0, 63, 5], dtype=torch.int32, device="cuda")
    eager, lengths = dec.caches(30), start.clone()
    want = []
    for x in xs:
        want.append(dec.step(x, eager, bt, lengths))
        lengths += 1
    caches, lengths, x = dec.caches(30), start.clone(), xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dec.step(x, caches, bt, lengths)
    for i in range(6):
        x.copy_(xs[i])
        graph.replay()
        assert torch.equal(y, want[i])
        lengths += 1
    for a, b in zip(eager, caches):
        assert torch.equal(a.k_codes, b.k_codes) and torch.equal(a.v_scale.view(torch.uint8), b.v_scale.view(torch.uint8))


def test_refusals():
    from voyager_b200.decode import CachedDecoder
    from voyager_b200.decoder import DecoderConfig, init_weights

    cfg = DecoderConfig(layers=1, hidden=512, heads=8, ffn=128)
    with pytest.raises(ValueError):
        CachedDecoder(cfg, init_weights(cfg, 0, "cuda"), cache_bits=5)
