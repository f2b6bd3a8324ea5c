"""The cached decoder: its operators run together, against a float32
computation of the same layers on unquantized weights, and decoding token by
token against the prompt in one step.

Tolerances.  An E4M3 rounding is at most 2^-4 relative, 2.6 % rms; a linear has
two such operands (3.7 %), and about six quantized stages lie on a layer's way
(q/k/v, the cache, o, gate/up, the activation, down), each at random: 9 % of
what the layers add to the residual stream; 15 % is allowed.  Token by token
the operands are the prompt's but for the float order of sums and for codes
that lay below 2^-9 of a block's scale: single bf16 roundings (0.4 %) that move
a code now and then; 3 % of the layers' sum is allowed."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _setup():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    import voyager_b200  # noqa: F401

    yield


def _decoder(kv_heads, head_dim, heads=8, layers=2):
    from voyager_b200.decode import CachedDecoder
    from voyager_b200.decoder import DecoderConfig, init_weights

    cfg = DecoderConfig(layers=layers, hidden=heads * head_dim, heads=heads, ffn=1408)
    w = init_weights(cfg, 3, "cuda")
    return cfg, w, CachedDecoder(cfg, w, kv_heads=kv_heads, max_positions=640)


def _float32(cfg, weights, kv_heads, x):
    """The layers on x [S, hidden] of one sequence, in float32."""
    from voyager_b200.decoder import apply_rope, rope_tables

    S, D = x.shape[0], cfg.head_dim
    cos, sin = rope_tables(S, D, cfg.rope_theta, x.device, torch.float32)
    kv = kv_heads * D
    h = x.float()
    for w in weights:
        w = {n: t.float() for n, t in w.items()}

        def norm(t, g):
            return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + cfg.eps) * g

        n = norm(h, w["ln1"])
        q, k, v = (n @ m.T for m in (w["q"], w["k"][:kv], w["v"][:kv]))
        q, k, v = (t.view(1, S, -1, D).transpose(1, 2) for t in (q, k, v))
        q, k = apply_rope(q, cos, sin), apply_rope(k, cos, sin)
        k, v = (t.repeat_interleave(cfg.heads // kv_heads, 1) for t in (k, v))
        s = (q @ k.transpose(-1, -2)) / D ** 0.5
        s = s.masked_fill(torch.ones(S, S, dtype=torch.bool, device=x.device).triu(1), float("-inf"))
        h = h + (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(S, -1) @ w["o"].T
        n = norm(h, w["ln2"])
        h = h + (torch.nn.functional.silu(n @ w["gate"].T) * (n @ w["up"].T)) @ w["down"].T
    return h


@pytest.mark.parametrize("kv_heads,head_dim", [(8, 128), (2, 64)])
def test_prompt_and_steps(kv_heads, head_dim):
    cfg, weights, dec = _decoder(kv_heads, head_dim)
    g = torch.Generator(device="cuda").manual_seed(1)
    S, B = 150, 2
    x = torch.randn(B, S, cfg.hidden, generator=g, device="cuda").bfloat16()
    counts = torch.tensor([S, 97], dtype=torch.int32, device="cuda")
    bt = torch.randperm(20, generator=g, device="cuda")[:20].view(B, 10).int()
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    caches = dec.caches(20)
    y = dec.step(x, caches, bt, zero, counts)
    for b in range(B):
        n = int(counts[b])
        want = _float32(cfg, weights, kv_heads, x[b, :n]) - x[b, :n].float()
        got = y[b, :n].float() - x[b, :n].float()
        assert float((got - want).norm() / want.norm()) < 0.15
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
    got = torch.cat(steps, 1)
    new = lengths[:, None] + torch.arange(40, device="cuda")
    base = x[rows, new].float()
    want = y[rows, new].float() - base
    assert float((got.float() - base - want).norm() / want.norm()) < 0.03


def test_step_in_a_graph():
    """A captured step replays with the plan advanced in place."""
    cfg, _, dec = _decoder(4, 64)
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
        assert torch.equal(a.k_codes.view(torch.uint8), b.k_codes.view(torch.uint8))


def test_refusals():
    from voyager_b200.decode import CachedDecoder
    from voyager_b200.decoder import DecoderConfig, init_weights

    cfg = DecoderConfig(layers=1, hidden=512, heads=8, ffn=128)
    w = init_weights(cfg, 0, "cuda")
    with pytest.raises(ValueError):
        CachedDecoder(cfg, w, kv_heads=3)
    with pytest.raises(ValueError):
        CachedDecoder(DecoderConfig(layers=1, hidden=512, heads=16, ffn=128), w)
