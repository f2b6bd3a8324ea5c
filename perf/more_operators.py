"""Cases of the 4-bit cache's operators and of the head norms: what is timed and compared.

Three operators of a decoder layer that decodes against a paged cache:

  norm     RMSNorm of every query and key head, rotary positions, and the new
           keys and values appended to a paged E4M3 cache, in one pass
  append   the same append (head norms or not) to a cache held in 4 bits: E2M1
           codes with one E4M3 scale for every 16 columns of a token, and the
           codes of the pool read back as values
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
BLOCK = 16           # columns of a token that share a scale in the 4-bit cache
QMAX = 448.0         # the largest E4M3 value
LEAST = 2.0 ** -9    # the smallest E4M3 value above 0: the smallest scale
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------------------
# cases
def listed():
    return [
        # one sequence decoding, a model with normalised heads: the smallest call
        {"name": "norm_one_token", "op": "norm", "B": 1, "T": 1, "L": 1000, "Hkv": 8, "G": 4, "D": 128,
         "page": 64, "rot": 128, "interleaved": False, "dtype": "bf16", "ragged": False},
        # a few drafted tokens of a batch of unequal lengths, half of each head turned, pairs side by side
        {"name": "norm_drafts", "op": "norm", "B": 64, "T": 5, "L": 900, "Hkv": 4, "G": 5, "D": 64,
         "page": 32, "rot": 32, "interleaved": True, "dtype": "f32", "ragged": True},
        # prompts of 2048 tokens written to the cache
        {"name": "norm_prompt", "op": "norm", "B": 8, "T": 2048, "L": 77, "Hkv": 8, "G": 4, "D": 128,
         "page": 64, "rot": 128, "interleaved": False, "dtype": "bf16", "ragged": False},
        # one sequence decoding into 4 bits
        {"name": "append_one_token", "op": "append", "B": 1, "T": 1, "L": 1000, "Hkv": 8, "G": 4, "D": 128,
         "page": 64, "rot": 128, "interleaved": False, "dtype": "bf16", "norm": False, "ragged": False},
        # a decoding batch of unequal lengths with normalised heads
        {"name": "append_batch", "op": "append", "B": 96, "T": 1, "L": 30000, "Hkv": 8, "G": 4, "D": 128,
         "page": 64, "rot": 64, "interleaved": False, "dtype": "bf16", "norm": True, "ragged": True},
        # prompts of 2048 tokens, every head with its own keys
        {"name": "append_prompt", "op": "append", "B": 8, "T": 2048, "L": 77, "Hkv": 32, "G": 1, "D": 128,
         "page": 64, "rot": 128, "interleaved": False, "dtype": "bf16", "norm": False, "ragged": False},
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
        # a piece of a long prompt over what the cache holds of it already
        {"name": "attend_chunk", "op": "attend", "B": 1, "T": 500, "L": 16011, "Hkv": 8, "G": 5, "D": 128,
         "page": 64, "ragged": False},
        # whole prompts over themselves: bound by the tensor cores
        {"name": "attend_prompt", "op": "attend", "B": 4, "T": 2048, "L": 0, "Hkv": 8, "G": 4, "D": 128,
         "page": 64, "ragged": False},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "append", "attend", "attend"])
    Hkv = rng.choice([1, 2, 4, 8, 8, 16, 32])
    G = rng.choice([1, 2, 4, 4, 5, 8] if Hkv <= 8 else [1, 2])
    D = rng.choice([64, 128, 128])
    page = rng.choice([32, 64, 64, 128])
    if op != "attend":
        T = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 2, 2048)])
        B = _log(rng, 1, max(1, min(128, 8 * 2048 * 96 * 128 // (T * (G + 2) * Hkv * D))))
        case = {"op": op, "B": B, "T": T, "L": _log(rng, 1, 4000 if op == "norm" else 60000) - 1, "Hkv": Hkv, "G": G,
                "D": D, "page": page, "rot": rng.choice([D, D, D // 2, D // 4]), "interleaved": rng.random() < 0.4,
                "dtype": rng.choice(["bf16", "bf16", "f32"] if T * B <= 4096 else ["bf16"]),
                "ragged": rng.random() < 0.6}
        if op == "append":
            case["norm"] = rng.random() < 0.5
        return case
    T = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 16, 2048)])
    L = _log(rng, 1, 131000) - 1
    if T > 16:
        L = min(L, 4 * 8 * 4 * 2048 * 2048 // (T * Hkv * G) // 2)
    # bytes of the cache for few rows, scores for many
    B = _log(rng, 1, max(1, min(64, 4 * 131000 * 8 * 128 // ((L + T) * Hkv * D),
                                4 * 8 * 4 * 2048 * 2048 // ((L + T) * T * Hkv * G))))
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


def _rotary_table(positions, rot, theta=10000.0, factor=4.0):
    """cos and sin of every pair's angle, float32 [positions, rot / 2, 2]; positions stretched
    linearly by `factor` for contexts longer than the model's own."""
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] / factor * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def _paged(case, gen, kept=False):
    """A cache's plan: which page holds which block of tokens; -1 past a sequence's last page.
    `kept`: only the pages that the new tokens touch are in the pool (the rest of each sequence
    lies elsewhere: -1 too)."""
    B, page = case["B"], case["page"]
    held, new = _lengths(case)
    width = max(1, -(-(case["L"] + case["T"]) // page))
    i32 = dict(dtype=torch.int32, device="cuda")
    h, n = torch.tensor(held, **i32), torch.tensor(new, **i32)
    at = torch.arange(width, device="cuda")[None]
    in_use = at < ((h + n + page - 1) // page)[:, None]
    if kept:
        in_use &= at >= (h // page)[:, None]
    pages = (sum(-(-(a + b) // page) - (a // page if kept else 0) for a, b in zip(held, new)) if kept else B * width) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    rank = (in_use.flatten().cumsum(0) - 1).clamp(min=0) if kept else torch.arange(B * width, device="cuda")
    table = torch.where(in_use, order[rank].reshape(B, width), -1).int().contiguous()
    return {"table": table, "held": h, "new": n if case["ragged"] else None, "pages": pages}


def _quantized(val, factor):
    """Values [.., D] and a factor that broadcasts to [.., 1] -> packed E2M1 codes uint8
    [.., D / 2] (the even column in the low half) and E4M3 scales [.., D / 16]."""
    b = val.unflatten(-1, (-1, BLOCK))
    scale = (b.abs().amax(-1) / (6.0 * factor)).clamp(LEAST, QMAX).to(E4M3)
    y = b / (scale.float() * factor)[..., None]
    a = y.abs()
    code = (a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = torch.where(y < 0, code + 8, code).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _cache4(case, gen, pages):
    """A pool of pages of normal values, some columns ten times the others', in 4 bits."""
    Hkv, page, D = case["Hkv"], case["page"], case["D"]
    st = {}
    for n, size in (("k", 1.0), ("v", 0.6)):
        st[n + "_factor"] = size * (0.05 + 0.1 * torch.rand(Hkv, generator=gen, device="cuda"))
        codes = torch.empty((pages, Hkv, page, D // 2), dtype=torch.uint8, device="cuda")
        scale = torch.empty((pages, Hkv, page, D // BLOCK), dtype=E4M3, device="cuda")
        wide = size * torch.exp(0.6 * _normal(gen, Hkv, 1, D))
        for lo in range(0, pages, step := max(1, (1 << 26) // (Hkv * page * D))):
            hi = min(pages, lo + step)
            c, s = _quantized(_normal(gen, hi - lo, Hkv, page, D) * wide, st[n + "_factor"][:, None, None])
            codes[lo:hi], scale[lo:hi] = c, s
        st[n + "_codes"], st[n + "_scale"] = codes, scale
    return st


def _cache8(case, gen, pages):
    """A pool of pages in E4M3 with a power-of-two scale for each page and head."""
    Hkv, page, D = case["Hkv"], case["page"], case["D"]
    st = {}
    for n in ("k", "v"):
        st[n + "_codes"] = (_normal(gen, pages, Hkv, page, D) * 100.0).clamp_(-QMAX, QMAX).to(E4M3)
        st[n + "_scale"] = torch.exp2(torch.randint(-8, -4, (pages, Hkv), generator=gen, device="cuda").float())
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, T, D, Hkv, page = case["B"], case["T"], case["D"], case["Hkv"], case["page"]
    H = Hkv * case["G"]
    st = {"case": case, "op": case["op"]}
    st.update(_paged(case, gen, kept=case["op"] == "append"))
    if case["op"] != "attend":
        st.update((_cache8 if case["op"] == "norm" else _cache4)(case, gen, st["pages"]))
        dt = TYPES[case["dtype"]]
        qkv = _normal(gen, B, T, H + 2 * Hkv, D).to(dt)  # one fused projection
        st["q"], st["k"], st["v"] = qkv.split([H, Hkv, Hkv], 2)
        normed = case["op"] == "norm" or case["norm"]
        st["qn"], st["kn"] = ((1.0 + 0.2 * _normal(gen, D)).to(dt) if normed else None for _ in range(2))
        st["rotary"] = _rotary_table(st["table"].shape[1] * page, case["rot"])
        return st
    st.update(_cache4(case, gen, st["pages"]))
    st["q"] = _normal(gen, B, T, H, D).bfloat16()
    # slots that no token has been written to hold whatever was there: here scales of NaN
    end = (st["held"] + (st["new"] if st["new"] is not None else T)).long()
    some = (end % page > 0).nonzero()[:, 0]
    last = st["table"][some, (end[some] // page)].long()
    stale = torch.arange(page, device="cuda")[None] >= (end[some] % page)[:, None]
    for n in ("k_scale", "v_scale"):
        raw = st[n].view(torch.uint8)
        raw[last] = torch.where(stale[:, None, :, None], 0x7F, raw[last]).to(torch.uint8)
    return st


# ---------------------------------------------------------------------------
# the operators in their plain form
def _normed(x, weight):
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()


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


def _plain_turn(st):
    """The turned queries in their type, the turned keys in 32 bits."""
    T = st["q"].shape[1]
    pos = (st["held"].long()[:, None] + torch.arange(T, device="cuda")).clamp(max=st["rotary"].shape[0] - 1)
    cs, flag = st["rotary"][pos], st["case"]["interleaved"]
    q = _rotated(_normed(st["q"].float(), st["qn"]), cs, flag)
    if st["new"] is not None:  # padding tokens have no query
        q = torch.where((torch.arange(T, device="cuda") < st["new"][:, None])[..., None, None], q, 0.0)
    return q.to(st["q"].dtype), _rotated(_normed(st["k"].float(), st["kn"]), cs, flag)


def _block_scale(amax):
    """The least power of two s in [2^-100, 2^120] with amax / s <= 448 (= 1.75 * 2^8)."""
    m, e = torch.frexp(amax)  # amax = m * 2^e, 0.5 <= m < 1
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.exp2(torch.where(amax > 0, e, -100).clamp(-100, 120).float())


def _plain_append8(st, new, codes, scale):
    """Values new [B, T, Hkv, D] written to the E4M3 cache after the tokens that it holds."""
    B, T, Hkv, D = new.shape
    page, held, table = codes.shape[2], st["held"].long(), st["table"]
    count = st["new"].long() if st["new"] is not None else torch.full_like(held, T)
    W = (T - 1) // page + 2  # pages that T tokens can touch
    at = (held // page)[:, None] + torch.arange(W, device="cuda")  # [B, W]
    touched = (at * page < (held + count)[:, None]) & (count > 0)[:, None]
    ids = torch.where(touched, table.gather(1, at.clamp(max=table.shape[1] - 1)).long(), 0)
    pos = (at[..., None] * page + torch.arange(page, device="cuda")).reshape(B, -1)  # [B, W * page]
    t = pos - held[:, None]
    is_new = ((t >= 0) & (t < count[:, None])).reshape(B, W, 1, page, 1)
    is_old = (t < 0).reshape(B, W, 1, page, 1)
    val = new.gather(1, t.clamp(0, T - 1)[..., None, None].expand(-1, -1, Hkv, D))
    val = val.reshape(B, W, page, Hkv, D).transpose(2, 3)  # [B, W, Hkv, page, D]
    need = _block_scale(torch.where(is_new, val.abs(), 0.0).amax((-1, -2)))
    was = scale[ids]
    s = torch.where((at * page < held[:, None])[..., None], torch.maximum(need, was), need)
    raw = codes.view(torch.uint8)[ids]
    kept = (raw.view(E4M3).float() * (was / s)[..., None, None]).to(E4M3)
    fresh = (val / s[..., None, None]).clamp(-QMAX, QMAX).to(E4M3)
    out = torch.where(is_new, fresh.view(torch.uint8), torch.where(is_old, kept.view(torch.uint8), raw))
    codes.view(torch.uint8)[ids[touched]] = out[touched]
    scale[ids[touched]] = s[touched]


def _plain_norm(st):
    q, k = _plain_turn(st)
    _plain_append8(st, k, st["k_codes"], st["k_scale"])
    _plain_append8(st, st["v"].float(), st["v_codes"], st["v_scale"])
    return q, st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"]


def _pairs():
    """The two values of each byte of E2M1 codes, [256, 2]."""
    v = torch.tensor(E2M1 + tuple(-x for x in E2M1), device="cuda")
    b = torch.arange(256, device="cuda")
    return torch.stack([v[b & 15], v[b >> 4]], -1)


def _plain_append4(st):
    q, k = _plain_turn(st)
    B, T = q.shape[:2]
    page, held = st["k_codes"].shape[2], st["held"].long()
    pos = held[:, None] + torch.arange(T, device="cuda")
    count = st["new"].long() if st["new"] is not None else torch.full_like(held, T)
    live = torch.arange(T, device="cuda") < count[:, None]
    pid = st["table"].gather(1, (pos // page).clamp(max=st["table"].shape[1] - 1)).long()[live]
    slot = (pos % page)[live]
    for n, val in (("k", k), ("v", st["v"].float())):
        codes, scale = _quantized(val[live], st[n + "_factor"][:, None])
        st[n + "_codes"][pid, :, slot] = codes
        st[n + "_scale"].view(torch.uint8)[pid, :, slot] = scale.view(torch.uint8)
    lut = _pairs().to(E4M3).view(torch.uint8)
    k, v = (lut[st[n + "_codes"].int()].flatten(-2).view(E4M3) for n in "kv")
    return q, k, v, st["k_scale"], st["v_scale"]


def _plain_attend(st):
    B, T, H, D = st["q"].shape
    table = st["table"].clamp(min=0).long()
    Hkv, page = st["k_codes"].shape[1:3]
    count = st["new"] if st["new"] is not None else torch.full_like(st["held"], T)
    end = (st["held"] + count)[:, None, None]
    keys = torch.arange(table.shape[1] * page, device="cuda")
    qpos = st["held"][:, None] + torch.arange(T, device="cuda")  # [B, T]
    seen = (keys <= qpos[..., None]) & (keys < end) & (torch.arange(T, device="cuda")[None] < count[:, None])[..., None]
    lut = _pairs()

    def whole(n):
        x = lut[st[n + "_codes"][table].int()].flatten(-2)  # [B, width, Hkv, page, D]
        s = st[n + "_scale"].view(torch.uint8)[table].view(E4M3).float() * st[n + "_factor"][:, None, None]
        x = (x.unflatten(-1, (-1, BLOCK)) * s[..., None]).flatten(-2)
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
    from voyager_b200 import kvcache

    return kvcache


def run(state):
    op, st = state["op"], state
    if not own:
        return {"norm": _plain_norm, "append": _plain_append4, "attend": _plain_attend}[op](st)
    kvcache = _package()
    held = (st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"])
    cache = kvcache.KVCache(*held) if op == "norm" else kvcache.KVCache4(*held, st["k_factor"], st["v_factor"])
    if op == "attend":
        return kvcache.attend(st["q"], cache, st["table"], st["held"], counts=st["new"])
    q = kvcache.rope_append(st["q"], st["k"], st["v"], st["rotary"], cache, st["table"], st["held"],
                            counts=st["new"], interleaved=st["case"]["interleaved"], q_norm=st["qn"],
                            k_norm=st["kn"], eps=EPS)
    k, v = held[:2] if op == "norm" else kvcache.unpack(cache)
    return q, k, v, st["k_scale"], st["v_scale"]


def work(case):
    held, new = _lengths(case)
    Hkv, G, D, page = case["Hkv"], case["G"], case["D"], case["page"]
    if case["op"] != "attend":
        n, b = sum(new), {"bf16": 2, "f32": 4}[case["dtype"]]
        # the heads read once, q written in its type, k and v as codes, each token's angles
        four = case["op"] == "append"
        moved = n * Hkv * D * (b * (G + 2) + b * G + 2 * (1 / 2 + 1 / 16 if four else 1)) + n * case["rot"] * 4
        if four:  # the pool's codes read, their values written
            pages = 3 + sum(-(-(h + c) // page) - h // page for h, c in zip(held, new))
            moved += pages * Hkv * page * D * 2 * (1 / 2 + 1)
        return {"bytes": moved, "flops": n * Hkv * (3 * case["rot"] * (G + 1) + 4 * D * (G + 2))}
    keys = sum(h + c for h, c in zip(held, new) if c)
    rows = sum(c * (h + (c + 1) / 2) for h, c in zip(held, new))
    return {"bytes": keys * Hkv * 2 * (D / 2 + D / BLOCK) + 4 * case["B"] * case["T"] * Hkv * G * D,
            "flops": 4 * rows * Hkv * G * D}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
def _e4m3_64(x):
    """float64 values rounded to the nearest E4M3 value (ties to even), saturating."""
    e = torch.frexp(x.abs().clamp(min=1e-300))[1].double() - 1
    step = torch.exp2(e.clamp(min=-6) - 3)
    return ((x / step).round() * step).clamp(-QMAX, QMAX)


def _e2m1_64(x):
    """float64 values rounded to the nearest E2M1 value (ties to the even code), saturating."""
    a = x.abs().clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0)).double()
    return torch.copysign((a / step).round() * step, x)


def _turned_64(st, n, i, h, c, case):
    """Sequence i's new heads of "q" or "k", normalised and turned, [c, heads, D]."""
    x, w = st[n][i, :c].double(), st[n + "n"]
    if w is not None:
        x = w.double() * x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    half = torch.arange(case["rot"] // 2, device="cuda")
    a, b = (2 * half, 2 * half + 1) if case["interleaved"] else (half, half + case["rot"] // 2)
    turn = st["rotary"][h:h + c].double()
    r = torch.complex(x[..., a], x[..., b]) * torch.complex(turn[..., 0], turn[..., 1])[:, None]
    x[..., a], x[..., b] = r.real, r.imag
    return x


def _exact_append(st, case):
    page, four = case["page"], case["op"] == "append"
    held, new = _lengths(case)
    q_out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    table, scales, codes = st["table"].tolist(), {}, {}
    for n in "kv":
        scales[n], raw = st[n + "_scale"].double(), st[n + "_codes"]
        if four:
            raw = torch.stack([raw & 15, raw >> 4], -1).flatten(-2).long()
            raw = torch.tensor([s * x for s in (1.0, -1.0) for x in E2M1], device="cuda")[raw]
        codes[n] = raw.double()
    for i, (h, c) in enumerate(zip(held, new)):
        if not c:
            continue
        q_out[i, :c] = _turned_64(st, "q", i, h, c, case)
        vals = {"k": _turned_64(st, "k", i, h, c, case), "v": st["v"][i, :c].double()}
        for p in range(h // page, (h + c - 1) // page + 1):
            lo, hi = max(h, p * page), min(h + c, (p + 1) * page)
            old, pid, into = max(0, h - p * page), table[i][p], slice(lo - p * page, hi - p * page)
            for n in "kv":
                x = vals[n][lo - h:hi - h].transpose(0, 1)  # [Hkv, tokens, D]
                if four:
                    f = st[n + "_factor"].double()[:, None, None]
                    b = x.reshape(*x.shape[:2], -1, BLOCK)
                    s = _e4m3_64(b.abs().max(-1).values / 6.0 / f).clamp(min=LEAST)
                    codes[n][pid, :, into] = _e2m1_64(b / (s * f)[..., None]).reshape(x.shape)
                    scales[n][pid, :, into] = s
                    continue
                top = x.abs().amax((1, 2)) / QMAX
                s = torch.exp2(torch.ceil(torch.log2(top.clamp(min=2.0 ** -100))))
                was = scales[n][pid]
                if old:
                    s = torch.maximum(s, was)
                    codes[n][pid, :, :old] = _e4m3_64(codes[n][pid, :, :old] * (was / s)[:, None, None])
                codes[n][pid, :, into] = _e4m3_64(x / s[:, None, None])
                scales[n][pid] = s
    return q_out, codes["k"], codes["v"], scales["k"], scales["v"]


def _exact_attend(st, case):
    Hkv, G, D = case["Hkv"], case["G"], case["D"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    value = torch.tensor([s * x for s in (1.0, -1.0) for x in E2M1], dtype=torch.float64, device="cuda")
    for i, (h, c) in enumerate(zip(*_lengths(case))):
        if not c:
            continue
        ids = st["table"][i, :-(-(h + c) // case["page"])].long()
        for g in range(Hkv):
            dense = []
            for n in "kv":
                raw = st[n + "_codes"][ids, g].reshape(-1, D // 2)[:h + c].long()
                x = torch.empty((h + c, D), dtype=torch.float64, device="cuda")
                x[:, 0::2], x[:, 1::2] = value[raw % 16], value[raw // 16]
                s = st[n + "_scale"].view(torch.uint8)[ids, g].view(E4M3).double().reshape(-1, D // BLOCK)[:h + c]
                dense.append(x * s.repeat_interleave(BLOCK, 1) * st[n + "_factor"][g].double())
            for lo in range(0, c, 512):
                t = torch.arange(lo, min(c, lo + 512), device="cuda")
                x = st["q"][i, t, g * G:(g + 1) * G].double()
                s = torch.einsum("tgd,kd->tgk", x, dense[0]) / D ** 0.5
                late = torch.arange(h + c, device="cuda") > h + t[:, None]
                out[i, t, g * G:(g + 1) * G] = torch.softmax(s.masked_fill(late[:, None], -math.inf), -1) @ dense[1]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_attend(st, case) if case["op"] == "attend" else _exact_append(st, case)
