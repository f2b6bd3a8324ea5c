"""E4M3 activations and weights with float32 scales per block of 128.

Activations [.., K] carry one scale per 128 columns of a row, weights [N, K]
one per 128 x 128 block.  These are the operands of a decoding step beside the
MXFP8 ones of ``quantize_mx``; codes are ``torch.float8_e4m3fn`` tensors.

  rmsnorm_quantize  (x + residual) -> RMSNorm -> codes, scales (and x + residual)
  quantize          x -> codes, scales
  quantize_weight   [N, K] -> codes, scales, once per weight
  linear            codes x weight codes -> bfloat16, on the tensor cores
"""

from typing import Optional, Tuple

import torch

from voyager_b200 import _lib
from voyager_b200._launch import call

BLOCK = 128
E4M3 = torch.float8_e4m3fn
QMAX = 448.0
_DTYPES = {torch.bfloat16: _lib.VQ_BF16, torch.float32: _lib.VQ_F32}


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """t as [rows, cols] with dense rows (a copy only where a view cannot be)."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    return t if t.stride(1) == 1 or cols == 1 else t.contiguous()


def _norm_quantize(x, residual, weight, eps, what):
    dtype = x.dtype
    code = _DTYPES.get(dtype)
    if code is None:
        raise NotImplementedError(f"{what}: bfloat16 or float32, not {dtype}")
    if not x.is_cuda:
        raise NotImplementedError(f"{what}: the CUDA kernel needs CUDA tensors")
    shape, index = x.shape, x.get_device()
    if not shape or shape[-1] == 0:
        raise ValueError(f"{what}: x needs a last dimension to normalise, got {tuple(shape)}")
    cols = shape[-1]
    x2 = _rows(x, cols)
    rows, ldx = x2.shape[0], max(x2.stride(0), cols)
    w = r = h = hidden = None
    ldr = 0
    if weight is not None:
        if weight.dtype != dtype or weight.get_device() != index or weight.shape != (cols,):
            raise ValueError(f"{what}: weight must be {dtype} [{cols}] on {x.device}")
        if weight.stride(0) != 1:
            weight = weight.contiguous()
        w = weight.data_ptr()
    if residual is not None:
        if residual.dtype != dtype or residual.get_device() != index or residual.shape != shape:
            raise ValueError(f"{what}: residual must be {dtype} {tuple(shape)} on {x.device}")
        residual = _rows(residual, cols)
        r, ldr = residual.data_ptr(), max(residual.stride(0), cols)
        hidden = x.new_empty(shape)
        h = hidden.data_ptr()
    codes = x.new_empty(shape, dtype=E4M3)
    scale = x.new_empty(shape[:-1] + ((cols + BLOCK - 1) // BLOCK,), dtype=torch.float32)
    call(_lib.load().vq_norm_quantize_fp8, index, what, x2.data_ptr(), ldx, r, ldr, w, code, rows, cols,
         eps, codes.data_ptr(), scale.data_ptr(), h)
    return codes, scale, hidden


def rmsnorm_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                     residual: Optional[torch.Tensor] = None
                     ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """``y = h * rsqrt(mean(h^2) + eps) * weight`` with ``h = x + residual`` in
    float32, quantized per 128 columns: ``(codes, scale, hidden)``, scale
    float32 [.., ceil(K / 128)], hidden = h in x's type (None without a
    residual).  x bfloat16 or float32 [.., K], any K; the norm is that of the
    unrounded sum."""
    return _norm_quantize(x, residual, weight, eps, "rmsnorm_quantize")


def quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [.., K] -> (codes, scale): ``scale = max|x| / 448`` per 128 columns (1
    where that is 0), ``codes = E4M3(x / scale)``."""
    return _norm_quantize(x, None, None, 0.0, "quantize")[:2]


def quantize_weight(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """w [N, K] -> (codes, scale [ceil(N / 128), ceil(K / 128)]), as
    ``quantize`` but over 128 x 128 blocks.  Done once per weight, by torch's
    elementwise ops."""
    if w.dim() != 2 or 0 in w.shape:
        raise ValueError(f"quantize_weight: a weight is [N, K], got {tuple(w.shape)}")
    N, K = w.shape
    f = torch.nn.functional.pad(w.float(), (0, -K % BLOCK, 0, -N % BLOCK))
    f = f.view(f.shape[0] // BLOCK, BLOCK, f.shape[1] // BLOCK, BLOCK)
    amax = f.abs().amax((1, 3))
    scale = torch.where(amax == 0, torch.ones_like(amax), amax / QMAX)
    codes = (f / scale[:, None, :, None]).clamp(-QMAX, QMAX).to(E4M3)
    return codes.view(codes.shape[0] * BLOCK, -1)[:N, :K].contiguous(), scale


def linear(codes: torch.Tensor, scale: torch.Tensor, w_codes: torch.Tensor, w_scale: torch.Tensor,
           bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``[.., K] x [N, K]^T (+ bias) -> [.., N]`` bfloat16 of the values that the
    codes and their block scales stand for: exact products, float32 sums, one
    rounding.  K a multiple of 16; any N and number of rows."""
    if codes.dtype != E4M3 or w_codes.dtype != E4M3:
        raise NotImplementedError("fp8block.linear takes float8_e4m3fn codes")
    if scale.dtype != torch.float32 or w_scale.dtype != torch.float32:
        raise NotImplementedError("fp8block.linear takes float32 scales")
    if not codes.is_cuda:
        raise NotImplementedError("fp8block.linear: the CUDA kernel needs CUDA tensors")
    index, shape, ws = codes.get_device(), codes.shape, w_codes.shape
    if len(ws) != 2 or not shape or shape[-1] != ws[1]:
        raise ValueError(f"fp8block.linear: {tuple(shape)} does not match a weight [N, K] {tuple(ws)}")
    N, K = ws
    if K == 0 or K % 16 or N == 0:
        raise ValueError(f"fp8block.linear: K = {K} must be a positive multiple of 16 and N = {N} positive")
    nk = (K + BLOCK - 1) // BLOCK
    lead = shape[:-1]
    if scale.shape != lead + (nk,) or w_scale.shape != ((N + BLOCK - 1) // BLOCK, nk):
        raise ValueError(f"fp8block.linear: scales {tuple(scale.shape)} and {tuple(w_scale.shape)} are not "
                         f"one per 128 columns and one per 128 x 128 block")
    if scale.get_device() != index or w_codes.get_device() != index or w_scale.get_device() != index:
        raise ValueError("fp8block.linear: operands on different devices")
    b = None
    if bias is not None:
        if bias.dtype != torch.bfloat16 or bias.shape != (N,) or bias.get_device() != index:
            raise ValueError(f"fp8block.linear: bias must be bfloat16 [{N}] on {codes.device}")
        bias = bias.contiguous()
        b = bias.data_ptr()
    codes, scale, w_codes, w_scale = codes.contiguous(), scale.contiguous(), w_codes.contiguous(), w_scale.contiguous()
    out = codes.new_empty(lead + (N,), dtype=torch.bfloat16)
    call(_lib.load().vq_linear_fp8_block, index, "fp8block.linear", codes.data_ptr(), scale.data_ptr(),
         w_codes.data_ptr(), w_scale.data_ptr(), b, codes.numel() // K, N, K, out.data_ptr(), N)
    return out
