"""Cases of the cached-decoding operators: what is timed and compared.

Four operators that a decoder layer runs in a row when it decodes against a
cache held in E4M3:

  norm     the residual's addition, RMSNorm, and E4M3 codes with one float32
           scale for every 128 columns of a row
  linear   those codes times an E4M3 weight with one float32 scale for every
           128 x 128 block, bfloat16 out
  rope     rotary positions of the query and key heads, and the new keys and
           values appended to a paged E4M3 cache whose blocks (one page of one
           head) each have a power-of-two scale
  attend   causal attention of the newest tokens over that cache

``own`` False: each operator in elementary torch operations in 32 bits.
``own`` True: the calls that a user of the package makes.
"""

import math
import os
import random
import sys

import torch

own = False

E4M3 = torch.float8_e4m3fn
BLOCK = 128          # columns of an activation, and rows and columns of a weight, per scale
QMAX = 448.0         # the largest E4M3 value
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# cases
def listed():
    return [
        # one decoded token at the decoder's hidden size: a call that is all latency
        {"name": "norm_one_token", "op": "norm", "R": 1, "C": 4096, "dtype": "bf16", "residual": True},
        # the layer norm over a prompt batch of 8 x 2048 tokens
        {"name": "norm_prompt", "op": "norm", "R": 16384, "C": 4096, "dtype": "bf16", "residual": True},
        # the fused q/k/v projection of one decoded token: the weight is read once
        {"name": "linear_one_token", "op": "linear", "M": 1, "N": 12288, "K": 4096},
        # a step's odd number of tokens, against a weight whose rows and columns fill no tile
        {"name": "linear_ragged", "op": "linear", "M": 333, "N": 5003, "K": 2000},
        # the gate and up projection of a prompt's 4096 tokens: bound by the tensor cores
        {"name": "linear_prompt", "op": "linear", "M": 4096, "N": 22016, "K": 4096},
        # one sequence decoding: the smallest call
        {"name": "rope_one_token", "op": "rope", "B": 1, "T": 1, "L": 1000, "Hkv": 8, "G": 4, "D": 128,
         "page": 64, "rot": 128, "interleaved": False, "dtype": "bf16", "ragged": False},
        # a decoding batch of unequal lengths, half of each head rotated, pairs side by side
        {"name": "rope_batch", "op": "rope", "B": 64, "T": 1, "L": 900, "Hkv": 8, "G": 4, "D": 128,
         "page": 64, "rot": 64, "interleaved": True, "dtype": "bf16", "ragged": True},
        # prompts of 2048 tokens written to the cache, every head with its own keys
        {"name": "rope_prompt", "op": "rope", "B": 8, "T": 2048, "L": 77, "Hkv": 32, "G": 1, "D": 128,
         "page": 64, "rot": 128, "interleaved": False, "dtype": "bf16", "ragged": False},
        # one sequence soon after its start: the smallest call
        {"name": "attend_short", "op": "attend", "B": 1, "T": 1, "L": 99, "Hkv": 8, "G": 4, "D": 128,
         "page": 64, "ragged": False},
        # a decoding batch of unequal lengths, some sequences still empty
        {"name": "attend_batch", "op": "attend", "B": 32, "T": 1, "L": 8192, "Hkv": 8, "G": 4, "D": 128,
         "page": 64, "ragged": True},
        # several drafted tokens of each sequence checked at once, heads of 64
        {"name": "attend_drafts", "op": "attend", "B": 6, "T": 5, "L": 20000, "Hkv": 4, "G": 7, "D": 64,
         "page": 32, "ragged": True},
        # few sequences with very long caches: the largest read
        {"name": "attend_long", "op": "attend", "B": 4, "T": 1, "L": 131000, "Hkv": 8, "G": 8, "D": 128,
         "page": 128, "ragged": False},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "rope", "attend"])
    if op == "norm":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        C = _log(rng, 64, 16384)
        C = C if rng.random() < 0.4 else (C + 127) // 128 * 128
        most = 16384 * 4096 // C // (1 if dtype == "bf16" else 2)
        return {"op": op, "R": _log(rng, 1, min(16384, most)), "C": C, "dtype": dtype,
                "residual": rng.random() < 0.7}
    if op == "linear":
        K = 16 * _log(rng, 4, 688)
        N = _log(rng, 64, 22016)
        N = N if rng.random() < 0.4 else (N + 127) // 128 * 128
        return {"op": op, "M": _log(rng, 1, min(4096, 4096 * 22016 * 4096 // (N * K))), "N": N, "K": K}
    Hkv = rng.choice([1, 2, 4, 8, 8, 16, 32])
    G = rng.choice([1, 2, 4, 4, 5, 8] if Hkv <= 8 else [1, 2])
    D = rng.choice([64, 128, 128])
    page = rng.choice([32, 64, 64, 128])
    if op == "rope":
        T = rng.choice([1, 1, 1, _log(rng, 2, 2048)])
        B = _log(rng, 1, max(1, min(128, 8 * 2048 * 96 * 128 // (T * (G + 2) * Hkv * D))))
        return {"op": op, "B": B, "T": T, "L": _log(rng, 1, 4000) - 1, "Hkv": Hkv, "G": G, "D": D, "page": page,
                "rot": rng.choice([D, D, D // 2]), "interleaved": rng.random() < 0.4,
                "dtype": rng.choice(["bf16", "bf16", "f32"] if T * B <= 4096 else ["bf16"]),
                "ragged": rng.random() < 0.6}
    T = rng.choice([1, 1, 1, _log(rng, 2, 12)])
    L = _log(rng, 1, 131000) - 1
    B = _log(rng, 1, max(1, min(64, 4 * 131000 * 8 * 128 // ((L + T) * Hkv * D * (1 if T * G <= 8 else 2)))))
    return {"op": op, "B": B, "T": T, "L": L, "Hkv": Hkv, "G": G, "D": D, "page": page,
            "ragged": rng.random() < 0.6}


def _lengths(case):
    """Tokens held in the cache before the step and new tokens, per sequence: a plan that the host
    has too.  Ragged: the first sequence is the longest, the last of three or more is empty."""
    B, L, T = case["B"], case["L"], case["T"]
    if not case["ragged"]:
        return [L] * B, [T] * B
    r = random.Random(1000003 * B + 131 * L + T)
    held = [L] + [r.randint(0, L) for _ in range(B - 1)]
    new = [T] + [r.randint(min(1, T), T) for _ in range(B - 1)]
    if B > 2:
        held[-1] = new[-1] = 0
    return held, new


# ---------------------------------------------------------------------------
# inputs
def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _codes(gen, *shape):
    """E4M3 codes of a normal distribution whose largest values come near 448."""
    out = torch.empty(shape, dtype=E4M3, device="cuda")
    for o in out.reshape(-1).split(1 << 28):
        o.copy_((_normal(gen, o.numel()) * 100.0).clamp_(-QMAX, QMAX))
    return out


def _rotary_table(positions, rot, theta=10000.0, factor=4.0):
    """cos and sin of every pair's angle, float32 [positions, rot / 2, 2]; positions stretched
    linearly by `factor` for contexts longer than the model's own."""
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] / factor * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def _paged(case, gen):
    """A cache's plan: which page holds which block of tokens; -1 past a sequence's last page."""
    B, page = case["B"], case["page"]
    held, new = _lengths(case)
    width = max(1, -(-(case["L"] + case["T"]) // page))
    pages = B * width + 3
    table = torch.randperm(pages, generator=gen, device="cuda")[:B * width].reshape(B, width).int()
    i32 = dict(dtype=torch.int32, device="cuda")
    held, new = torch.tensor(held, **i32), torch.tensor(new, **i32)
    used = (held + new + page - 1) // page
    table = torch.where(torch.arange(width, device="cuda")[None] < used[:, None], table, -1).contiguous()
    return {"table": table, "held": held, "new": new if case["ragged"] else None, "pages": pages}


def _cache(case, gen, pages):
    Hkv, page, D = case["Hkv"], case["page"], case["D"]
    st = {}
    for n in ("k", "v"):
        st[n + "_codes"] = _codes(gen, pages, Hkv, page, D)
        st[n + "_scale"] = torch.exp2(torch.randint(-8, -4, (pages, Hkv), generator=gen, device="cuda").float())
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": case, "op": case["op"]}
    if case["op"] == "norm":
        dt, R, C = TYPES[case["dtype"]], case["R"], case["C"]
        st["x"] = _normal(gen, R, C).to(dt)
        st["residual"] = (2.0 * _normal(gen, R, C)).to(dt) if case["residual"] else None
        st["weight"] = (1.0 + 0.1 * _normal(gen, C)).to(dt)
    elif case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        nk = -(-K // BLOCK)
        st["a"], st["w"] = _codes(gen, M, K), _codes(gen, N, K)
        st["sa"] = torch.rand((M, nk), generator=gen, device="cuda") * 0.01 + 0.002
        st["sw"] = torch.rand((-(-N // BLOCK), nk), generator=gen, device="cuda") * 1e-4 + 1e-5
        st["bias"] = _normal(gen, N).bfloat16()
    elif case["op"] == "rope":
        B, T, D, Hkv = case["B"], case["T"], case["D"], case["Hkv"]
        H = Hkv * case["G"]
        st.update(_paged(case, gen))
        st.update(_cache(case, gen, st["pages"]))
        qkv = _normal(gen, B, T, H + 2 * Hkv, D).to(TYPES[case["dtype"]])  # one fused projection
        st["q"], st["k"], st["v"] = qkv.split([H, Hkv, Hkv], 2)
        st["rotary"] = _rotary_table(st["table"].shape[1] * case["page"], case["rot"])
    else:
        B, T, D, Hkv, page = case["B"], case["T"], case["D"], case["Hkv"], case["page"]
        st.update(_paged(case, gen))
        st.update(_cache(case, gen, st["pages"]))
        st["q"] = _normal(gen, B, T, Hkv * case["G"], D).bfloat16()
        # slots that no token has been written to hold whatever was there: here NaN
        end = (st["held"] + (st["new"] if st["new"] is not None else T)).long()
        some = (end % page > 0).nonzero()[:, 0]
        last = st["table"][some, (end[some] // page)].long()
        stale = torch.arange(page, device="cuda")[None] >= (end[some] % page)[:, None]
        for n in ("k_codes", "v_codes"):
            raw = st[n].view(torch.uint8)
            raw[last] = torch.where(stale[:, None, :, None], 0x7F, raw[last]).to(torch.uint8)
    return st


# ---------------------------------------------------------------------------
# the operators in their plain form
def _plain_norm(st):
    x = st["x"].float()
    hidden = None
    if st["residual"] is not None:
        x = x + st["residual"].float()
        hidden = x.to(st["x"].dtype)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * st["weight"].float()
    R, C = y.shape
    y = torch.nn.functional.pad(y, (0, -C % BLOCK)).reshape(R, -1, BLOCK)
    amax = y.abs().amax(-1)
    scale = torch.where(amax == 0, torch.ones_like(amax), amax / QMAX)
    codes = (y / scale[..., None]).clamp(-QMAX, QMAX).to(E4M3).reshape(R, -1)[:, :C]
    return (codes, scale) if hidden is None else (codes, scale, hidden)


def _spread(codes, scale, rows):
    """The values of codes [R, K] with a scale for each `rows` x 128 block."""
    s = scale.repeat_interleave(rows, 0)[:codes.shape[0]].repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]
    return codes.float() * s


def _plain_linear(st):
    y = _spread(st["a"], st["sa"], 1) @ _spread(st["w"], st["sw"], BLOCK).T
    return (y + st["bias"].float()).bfloat16()


def _rotated(x, cs, interleaved):
    """x [B, T, heads, D] with the first rot columns turned by the angles cs [B, T, rot / 2, 2]."""
    rot = 2 * cs.shape[2]
    c, s = cs[:, :, None, :, 0], cs[:, :, None, :, 1]
    head, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([head, rest], -1)


def _block_scale(amax):
    """The least power of two s in [2^-100, 2^120] with amax / s <= 448 (= 1.75 * 2^8)."""
    m, e = torch.frexp(amax)  # amax = m * 2^e, 0.5 <= m < 1
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.exp2(torch.where(amax > 0, e, -100).clamp(-100, 120).float())


def _plain_append(st, new, codes, scale):
    """Values new [B, T, Hkv, D] written to the cache after the tokens that it holds."""
    B, T, Hkv, D = new.shape
    page, held, table = codes.shape[2], st["held"].long(), st["table"]
    count = st["new"].long() if st["new"] is not None else torch.full_like(held, T)
    W = (T - 1) // page + 2  # pages that T tokens can touch
    first = held // page
    at = first[:, None] + torch.arange(W, device="cuda")  # [B, W]
    touched = (at * page < (held + count)[:, None]) & (count > 0)[:, None]
    ids = table.gather(1, at.clamp(max=table.shape[1] - 1)).long()
    ids = torch.where(touched, ids, 0)
    pos = (at[..., None] * page + torch.arange(page, device="cuda")).reshape(B, -1)  # [B, W * page]
    t = pos - held[:, None]
    is_new = ((t >= 0) & (t < count[:, None])).reshape(B, W, 1, page, 1)
    is_old = (t < 0).reshape(B, W, 1, page, 1)
    val = new.gather(1, t.clamp(0, T - 1)[..., None, None].expand(-1, -1, Hkv, D))
    val = val.reshape(B, W, page, Hkv, D).transpose(2, 3)  # [B, W, Hkv, page, D]
    amax = torch.where(is_new, val.abs(), 0.0).amax((-1, -2))
    need = _block_scale(amax)
    has_old = (at * page < held[:, None])[..., None]
    was = scale[ids]
    s = torch.where(has_old, torch.maximum(need, was), need)
    raw = codes.view(torch.uint8)[ids]
    kept = (raw.view(E4M3).float() * (was / s)[..., None, None]).to(E4M3)
    fresh = (val / s[..., None, None]).clamp(-QMAX, QMAX).to(E4M3)
    out = torch.where(is_new, fresh.view(torch.uint8), torch.where(is_old, kept.view(torch.uint8), raw))
    codes.view(torch.uint8)[ids[touched]] = out[touched]
    scale[ids[touched]] = s[touched]


def _plain_rope(st):
    dt = st["q"].dtype
    T = st["q"].shape[1]
    pos = (st["held"].long()[:, None] + torch.arange(T, device="cuda")).clamp(max=st["rotary"].shape[0] - 1)
    cs = st["rotary"][pos]
    flag = st["case"]["interleaved"]
    q = _rotated(st["q"].float(), cs, flag)
    if st["new"] is not None:  # padding tokens have no query
        q = torch.where((torch.arange(T, device="cuda") < st["new"][:, None])[..., None, None], q, 0.0)
    _plain_append(st, _rotated(st["k"].float(), cs, flag), st["k_codes"], st["k_scale"])
    _plain_append(st, st["v"].float(), st["v_codes"], st["v_scale"])
    return q.to(dt), st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"]


def _plain_attend(st):
    B, T, H, D = st["q"].shape
    table = st["table"].clamp(min=0).long()
    Hkv, page = st["k_codes"].shape[1:3]
    count = st["new"] if st["new"] is not None else torch.full_like(st["held"], T)
    end = (st["held"] + count)[:, None, None]
    keys = torch.arange(table.shape[1] * page, device="cuda")
    qpos = st["held"][:, None] + torch.arange(T, device="cuda")  # [B, T]
    seen = (keys <= qpos[..., None]) & (keys < end) & (torch.arange(T, device="cuda")[None] < count[:, None])[..., None]

    def whole(n):
        x = st[n + "_codes"].view(torch.uint8)[table].view(E4M3).float() * st[n + "_scale"][table][..., None, None]
        x = x.transpose(1, 2).reshape(B, Hkv, -1, D)
        return torch.where((keys < end)[..., None], x, 0.0)

    q = st["q"].float().reshape(B, T, Hkv, H // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    s = (q @ whole("k").transpose(-1, -2) / math.sqrt(D)).reshape(B, Hkv, T, H // Hkv, -1)
    s = torch.where(seen[:, None, :, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    norm = p.sum(-1, keepdim=True)
    o = p.reshape(B, Hkv, T * (H // Hkv), -1) @ whole("v")
    o = o.reshape(B, Hkv, T, H // Hkv, D) / torch.where(norm == 0, 1.0, norm)
    return o.permute(0, 2, 1, 3, 4).reshape(B, T, H, D).bfloat16()


# ---------------------------------------------------------------------------
def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "voyager-compiler_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from voyager_b200 import fp8block, kvcache

    return fp8block, kvcache


def run(state):
    op, st = state["op"], state
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "rope": _plain_rope, "attend": _plain_attend}[op](st)
    fp8block, kvcache = _package()
    if op == "norm":
        codes, scale, hidden = fp8block.rmsnorm_quantize(st["x"], st["weight"], 1e-5, residual=st["residual"])
        return (codes, scale) if hidden is None else (codes, scale, hidden)
    if op == "linear":
        return fp8block.linear(st["a"], st["sa"], st["w"], st["sw"], bias=st["bias"])
    cache = kvcache.KVCache(st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"])
    if op == "rope":
        q = kvcache.rope_append(st["q"], st["k"], st["v"], st["rotary"], cache, st["table"], st["held"],
                                counts=st["new"], interleaved=st["case"]["interleaved"])
        return q, st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"]
    return kvcache.attend(st["q"], cache, st["table"], st["held"], counts=st["new"])


def work(case):
    if case["op"] == "norm":
        n, b = case["R"] * case["C"], {"bf16": 2, "f32": 4}[case["dtype"]]
        return {"bytes": n * (b * (3 if case["residual"] else 1) + 1) + case["C"] * b
                + case["R"] * -(-case["C"] // BLOCK) * 4, "flops": 8 * n}
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        nk = -(-K // BLOCK)
        return {"bytes": (M + N) * K + 4 * nk * (M + -(-N // BLOCK)) + 2 * M * N + 2 * N, "flops": 2 * M * N * K}
    held, new = _lengths(case)
    Hkv, G, D = case["Hkv"], case["G"], case["D"]
    if case["op"] == "rope":
        n, b = sum(new), {"bf16": 2, "f32": 4}[case["dtype"]]
        # the heads read once, q written in its type, k and v as codes, each token's angles
        return {"bytes": n * Hkv * D * (b * (G + 2) + b * G + 2) + n * case["rot"] * 4,
                "flops": n * Hkv * (3 * case["rot"] * (G + 1) + 4 * D)}
    keys = sum(h + c for h, c in zip(held, new) if c)
    blocks = sum(-(-(h + c) // case["page"]) for h, c in zip(held, new) if c)
    rows = sum(c * (h + (c + 1) / 2) for h, c in zip(held, new))
    return {"bytes": keys * Hkv * 2 * D + blocks * Hkv * 8 + 4 * case["B"] * case["T"] * Hkv * G * D,
            "flops": 4 * rows * Hkv * G * D}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
def _e4m3_64(x):
    """float64 values rounded to the nearest E4M3 value (ties to even), saturating; NaN stays."""
    e = torch.frexp(x.abs().clamp(min=1e-300))[1].double() - 1
    step = torch.exp2(e.clamp(min=-6) - 3)
    return torch.where(x.isnan(), x, ((x / step).round() * step).clamp(-QMAX, QMAX))


def _exact_norm(st):
    x = st["x"].double()
    if st["residual"] is not None:
        x = x + st["residual"].double()
    y = st["weight"].double() * x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-5).sqrt()
    codes, scales = torch.empty_like(y), []
    for c in range(0, y.shape[1], BLOCK):
        b = y[:, c:c + BLOCK]
        s = b.abs().max(-1, keepdim=True).values / QMAX
        s = torch.where(s > 0, s, 1.0)
        codes[:, c:c + BLOCK] = _e4m3_64(b / s)
        scales.append(s)
    out = (codes, torch.cat(scales, 1))
    return out if st["residual"] is None else out + (x,)


def _exact_linear(st):
    a, w = st["a"].double(), st["w"].double()
    y = st["bias"].double().expand(a.shape[0], -1).clone()
    for k in range(0, a.shape[1], BLOCK):
        ws = st["sw"][:, k // BLOCK].double().repeat_interleave(BLOCK)[:w.shape[0], None]
        y.addmm_(a[:, k:k + BLOCK] * st["sa"][:, k // BLOCK, None].double(), (w[:, k:k + BLOCK] * ws).T)
    return y


def _exact_rope(st, case):
    D, page, rot = case["D"], case["page"], case["rot"]
    T, H = st["q"].shape[1:3]
    held, new = _lengths(case)
    half = torch.arange(rot // 2, device="cuda")
    a, b = (2 * half, 2 * half + 1) if case["interleaved"] else (half, half + rot // 2)
    q_out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    codes = {n: st[n + "_codes"].double() for n in "kv"}
    scales = {n: st[n + "_scale"].double() for n in "kv"}
    table = st["table"].tolist()
    for i, (h, c) in enumerate(zip(held, new)):
        if not c:
            continue
        turn = st["rotary"][h:h + c].double()
        z = torch.complex(turn[..., 0], turn[..., 1])[:, None]
        vals = {}
        for n in "qk":
            x = st[n][i, :c].double()
            r = torch.complex(x[..., a], x[..., b]) * z
            x[..., a], x[..., b] = r.real, r.imag
            vals[n] = x
        q_out[i, :c] = vals["q"]
        vals["v"] = st["v"][i, :c].double()
        for p in range(h // page, (h + c - 1) // page + 1):
            lo, hi = max(h, p * page), min(h + c, (p + 1) * page)
            old, pid = max(0, h - p * page), table[i][p]
            for n in "kv":
                x = vals[n][lo - h:hi - h].transpose(0, 1)  # [Hkv, tokens, D]
                top = x.abs().amax((1, 2)) / QMAX
                s = torch.exp2(torch.ceil(torch.log2(top.clamp(min=2.0 ** -100))))
                was = scales[n][pid]
                if old:
                    s = torch.maximum(s, was)
                    codes[n][pid, :, :old] = _e4m3_64(codes[n][pid, :, :old] * (was / s)[:, None, None])
                codes[n][pid, :, lo - p * page:hi - p * page] = _e4m3_64(x / s[:, None, None])
                scales[n][pid] = s
    return q_out, codes["k"], codes["v"], scales["k"], scales["v"]


def _exact_attend(st, case):
    Hkv, G, D, page = case["Hkv"], case["G"], case["D"], case["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for i, (h, c) in enumerate(zip(*_lengths(case))):
        if not c:
            continue
        ids = st["table"][i, :-(-(h + c) // page)].long()
        for g in range(Hkv):
            k, v = ((st[n + "_codes"][:, g].view(torch.uint8)[ids].view(E4M3).double()
                     * st[n + "_scale"][ids, g, None, None].double()).reshape(-1, D)[:h + c] for n in "kv")
            x = st["q"][i, :c, g * G:(g + 1) * G].double()
            s = torch.einsum("tgd,kd->tgk", x, k) / D ** 0.5
            late = torch.arange(h + c, device="cuda") > h + torch.arange(c, device="cuda")[:, None]
            p = torch.softmax(s.masked_fill(late[:, None], -math.inf), -1)
            out[i, :c, g * G:(g + 1) * G] = p @ v
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(st)
    if case["op"] == "linear":
        return _exact_linear(st)
    return _exact_rope(st, case) if case["op"] == "rope" else _exact_attend(st, case)
