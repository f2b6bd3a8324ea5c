"""E4M3 activations and weights with float32 scales per block of 128.

Activations [.., K] carry one scale per 128 columns of a row, weights [N, K]
one per 128 x 128 block.  These are the operands of a decoding step beside the
MXFP8 ones of ``quantize_mx``; codes are ``torch.float8_e4m3fn`` tensors.  They
serve inference: a backward pass that reaches their outputs raises.

  rmsnorm_quantize  (x + residual) -> RMSNorm -> codes, scales (and x + residual)
  quantize          x -> codes, scales
  quantize_weight   [N, K] -> codes, scales, once per weight
  linear            codes x weight codes -> bfloat16, on the tensor cores
"""

from typing import Optional, Tuple

import torch

from voyager_b200._launch import native

BLOCK = 128
E4M3 = torch.float8_e4m3fn
QMAX = 448.0


def rmsnorm_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                     residual: Optional[torch.Tensor] = None
                     ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """``y = h * rsqrt(mean(h^2) + eps) * weight`` with ``h = x + residual`` in
    float32, quantized per 128 columns: ``(codes, scale, hidden)``, scale
    float32 [.., ceil(K / 128)], hidden = h in x's type (None without a
    residual).  x bfloat16 or float32 [.., K], any K; the norm is that of the
    unrounded sum."""
    if weight is None:  # to the binding: no norm
        raise TypeError("rmsnorm_quantize: weight must be a tensor")
    return native.norm_quantize(x, residual, weight, eps, "rmsnorm_quantize")


def quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [.., K] -> (codes, scale): ``scale = max|x| / 448`` per 128 columns (1
    where that is 0 in float32), ``codes = E4M3(x / scale)``."""
    return native.norm_quantize(x, None, None, 0.0, "quantize")[:2]


def quantize_weight(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """w [N, K] -> (codes, scale [ceil(N / 128), ceil(K / 128)]), as
    ``quantize`` but over 128 x 128 blocks.  Done once per weight, by torch's
    elementwise ops."""
    if w.dim() != 2 or 0 in w.shape:
        raise ValueError(f"quantize_weight: a weight is [N, K], got {tuple(w.shape)}")
    N, K = w.shape
    f = torch.nn.functional.pad(w.float(), (0, -K % BLOCK, 0, -N % BLOCK))
    f = f.view(f.shape[0] // BLOCK, BLOCK, f.shape[1] // BLOCK, BLOCK)
    scale = f.abs().amax((1, 3)) / QMAX
    scale = torch.where(scale == 0, 1.0, scale)
    codes = (f / scale[:, None, :, None]).clamp(-QMAX, QMAX).to(E4M3)
    return codes.view(codes.shape[0] * BLOCK, -1)[:N, :K].contiguous(), scale


def linear(codes: torch.Tensor, scale: torch.Tensor, w_codes: torch.Tensor, w_scale: torch.Tensor,
           bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``[.., K] x [N, K]^T (+ bias) -> [.., N]`` bfloat16 of the values that the
    codes and their block scales stand for: exact products, float32 sums, one
    rounding.  The product of an activation's and a weight's scale is formed in
    float32 (normal from 2^-126 to 2^128).  K a multiple of 16; any N and number
    of rows."""
    return native.linear(codes, scale, w_codes, w_scale, bias)
