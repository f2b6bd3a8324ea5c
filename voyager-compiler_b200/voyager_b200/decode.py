"""A decoder stack that decodes against a key / value cache in E4M3 or in 4 bits:
the worked example of the cached-decoding operators, on one GPU.

The layers are those of ``voyager_b200.decoder`` (RMSNorm, rotary attention,
SwiGLU; ``DecoderConfig``, ``init_weights``), with grouped key / value heads and
every linear on E4M3 codes with float32 scales per 128:

  norm -> q/k/v linear -> (head norms +) rotary + append -> attend -> quantize -> o linear
  (+ residual) norm -> gate/up linear -> SwiGLU -> quantize -> down linear

One ``step`` takes the new tokens of every sequence, a whole prompt or a
single token alike; nothing in it waits for the device, so a step can be
captured in a CUDA graph and replayed with the plan's tensors updated in place.

    dec = CachedDecoder(cfg, init_weights(cfg, 0, "cuda"), kv_heads=8, max_positions=4096)
    caches = dec.caches(pages=512)
    y = dec.step(x, caches, block_table, lengths)       # x [B, T, hidden]
    lengths += x.shape[1]
"""

from typing import Dict, List, Optional

import torch

from voyager_b200 import fp8block, kvcache
from voyager_b200.decoder import DecoderConfig


class CachedDecoder:
    """``weights`` as ``decoder.init_weights`` makes them ([out, in]; the first
    kv_heads * head_dim rows of "k" and "v" are used), quantized here once.  A
    layer that has "q_norm" or "k_norm" [head_dim] normalises its query or key
    heads before they turn.  ``cache_bits``: 8, or 4 for ``KVCache4``."""

    def __init__(self, cfg: DecoderConfig, weights: List[Dict[str, torch.Tensor]], *,
                 kv_heads: Optional[int] = None, max_positions: int = 4096, page: int = 64, cache_bits: int = 8, **rotary):
        if cache_bits not in (4, 8):
            raise ValueError(f"cache_bits {cache_bits} is not 4 or 8")
        self.cfg, self.page, self.cache_bits = cfg, page, cache_bits
        self.kv_heads = cfg.heads if kv_heads is None else kv_heads
        if self.kv_heads <= 0 or cfg.heads % self.kv_heads:
            raise ValueError(f"{cfg.heads} heads do not group over {self.kv_heads} kv heads")
        if cfg.head_dim not in kvcache.HEAD_DIMS:
            raise ValueError(f"head_dim {cfg.head_dim} is not one of {kvcache.HEAD_DIMS}")
        self.device = weights[0]["q"].device
        # whole pages, so that every block table up to max_positions is covered
        positions = (max_positions + page - 1) // page * page
        self.table = kvcache.rotary_table(positions, cfg.head_dim, cfg.rope_theta, device=self.device, **rotary)
        kv = self.kv_heads * cfg.head_dim
        self.layers = []
        for w in weights:
            q = fp8block.quantize_weight
            self.layers.append({
                "qkv": q(torch.cat([w["q"], w["k"][:kv], w["v"][:kv]])), "o": q(w["o"]),
                "gu": q(torch.cat([w["gate"], w["up"]])), "down": q(w["down"]),
                "ln1": w["ln1"], "ln2": w["ln2"],
                "q_norm": w.get("q_norm"), "k_norm": w.get("k_norm")})

    def caches(self, pages: int) -> List[kvcache.Cache]:
        """An empty cache of `pages` pages per layer, in 4 bits with factors of 1: keys or
        values of a layer whose blocks stay below 0.094 need smaller ones (``KVCache4``),
        written to its ``k_factor`` / ``v_factor`` before the first step."""
        kind = kvcache.KVCache if self.cache_bits == 8 else kvcache.KVCache4
        return [kind.empty(pages, self.kv_heads, self.cfg.head_dim, self.page, self.device) for _ in self.layers]

    @torch.no_grad()
    def step(self, x: torch.Tensor, caches: List[kvcache.Cache], block_table: torch.Tensor,
             lengths: torch.Tensor, counts: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The hidden states x [B, T, hidden] (bfloat16) of each sequence's new
        tokens -> the same after all layers; the caches then hold them too.  The
        plan (block_table, lengths, counts) as in ``voyager_b200.kvcache``; the
        outputs of tokens past counts are not meaningful."""
        cfg, H, Hkv, D = self.cfg, self.cfg.heads, self.kv_heads, self.cfg.head_dim
        B, T, _ = x.shape
        h, residual = x, None
        for w, cache in zip(self.layers, caches):
            codes, scale, total = fp8block.rmsnorm_quantize(h, w["ln1"], cfg.eps, residual)
            residual = h if total is None else total
            qkv = fp8block.linear(codes, scale, *w["qkv"]).view(B, T, H + 2 * Hkv, D)
            q, k, v = qkv.split([H, Hkv, Hkv], 2)
            q = kvcache.rope_append(q, k, v, self.table, cache, block_table, lengths, counts, q_norm=w["q_norm"],
                                    k_norm=w["k_norm"], eps=cfg.eps)
            o = kvcache.attend(q, cache, block_table, lengths, counts).view(B, T, H * D)
            h = fp8block.linear(*fp8block.quantize(o), *w["o"])
            codes, scale, residual = fp8block.rmsnorm_quantize(h, w["ln2"], cfg.eps, residual)
            gate, up = fp8block.linear(codes, scale, *w["gu"]).chunk(2, -1)
            h = fp8block.linear(*fp8block.quantize(torch.nn.functional.silu(gate) * up), *w["down"])
        return h + residual
