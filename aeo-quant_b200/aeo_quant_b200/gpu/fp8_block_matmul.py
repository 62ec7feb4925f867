"""Block-scaled FP8 matrix products on B200: e4m3 weights with one f32 scale
per 128 x 128 block, activations quantized per 128 values of a row.

* :func:`fp8_block_linear` — quantize the activation, then the GEMM;
* :func:`fp8_block_linear_prequantized` — the GEMM alone.

The weights come from ``gpu.quant.quantize_2d_to_fp8_block`` or a checkpoint
in the same format; ``bridges.gemma4.linear_fp8.LinearFP8Block`` is the
module around them and ``bridges.gemma4.moe_ops.fp8_block_experts`` the
routed experts' forward. The kernels are in ``csrc/fp8_block_gemm.cu``. The
reference's FP8 linear has one scale per row
(``bridges.gemma4.linear_fp8.fp8_linear``).

Forward only: the weights are frozen and the outputs carry no gradient.
"""
from __future__ import annotations

import torch

from .. import _capi as A
from .quant import FP8_BLOCK

_OUT_DT = {torch.bfloat16: A.BF16, torch.float32: A.F32}
_IN_DT = (torch.bfloat16, torch.float16, torch.float32)


def _check_weight(w_fp8: torch.Tensor, w_scale: torch.Tensor) -> tuple[int, int]:
    if w_fp8.ndim != 2:
        raise ValueError(f"w_fp8 must be 2D (N, K), got shape {tuple(w_fp8.shape)}")
    if w_fp8.dtype not in (torch.float8_e4m3fn, torch.uint8):
        raise ValueError(f"w_fp8 must be float8_e4m3fn, got {w_fp8.dtype}")
    N, K = w_fp8.shape
    want = (-(-N // FP8_BLOCK), -(-K // FP8_BLOCK))
    if w_scale.shape != want or w_scale.dtype != torch.float32:
        raise ValueError(f"w_scale must be float32 of shape {want} (one per {FP8_BLOCK} x {FP8_BLOCK} block), "
                         f"got {w_scale.dtype} {tuple(w_scale.shape)}")
    return N, K


def _check_out(out_dtype: torch.dtype, bias, N: int) -> int:
    if out_dtype not in _OUT_DT:
        raise ValueError(f"out_dtype must be torch.bfloat16 or torch.float32, got {out_dtype}")
    if bias is not None and (tuple(bias.shape) != (N,) or bias.dtype != torch.bfloat16):
        raise ValueError(f"bias must be bfloat16 of shape ({N},), got {bias.dtype} {tuple(bias.shape)}")
    return _OUT_DT[out_dtype]


def fp8_block_linear(x: torch.Tensor, w_fp8: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None = None, *,
                     out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x @ W^T + bias``: x (..., K) bfloat16, float16 or float32, quantized
    per 128 values of a row in the call; ``w_fp8`` (N, K) e4m3 with
    ``w_scale`` (ceil(N/128), ceil(K/128)) float32; optional bfloat16 bias.
    K must be a multiple of 16; N is free. Sums are f32, rounded once to
    ``out_dtype`` (bfloat16 or float32). Returns (..., N)."""
    N, K = _check_weight(w_fp8, w_scale)
    code = _check_out(out_dtype, bias, N)
    if x.dtype not in _IN_DT:
        raise ValueError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if x.shape[-1] != K:
        raise ValueError(f"input features {x.shape[-1]} != weight in_features {K}")
    dev = A.cuda_index(x, w_fp8, w_scale, bias)
    lib = A.load()
    with A.on_device(dev):
        x2 = x if x.ndim == 2 else x.reshape(-1, K)
        M = x2.shape[0]
        if M and (x2.stride(1) != 1 or (M > 1 and x2.stride(0) < K)):
            x2 = x2.contiguous()
        out = torch.empty((M, N), dtype=out_dtype, device=x.device)
        n = lib.aeoq_fp8_block_linear_workspace_size(M, N, K)
        ws = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
        if not w_fp8.is_contiguous():
            w_fp8 = w_fp8.contiguous()
        if not w_scale.is_contiguous():
            w_scale = w_scale.contiguous()
        if bias is not None:
            bias = bias.contiguous()
        A.check(lib.aeoq_fp8_block_linear(x2.data_ptr(), A.dtype_code(x.dtype), x2.stride(0) if M > 1 else K, M,
                                          w_fp8.data_ptr(), w_scale.data_ptr(), N, K, A.ptr(bias), out.data_ptr(),
                                          code, N, A.ptr(ws), n, A.err_ptr(dev), A.raw_stream(dev)))
    return out if x.ndim == 2 else out.reshape(*x.shape[:-1], N)


def fp8_block_linear_prequantized(x_fp8: torch.Tensor, x_scale: torch.Tensor, w_fp8: torch.Tensor,
                                  w_scale: torch.Tensor, bias: torch.Tensor | None = None, *,
                                  out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The product alone, for an activation that
    ``quantize_fp8_activation_blocks`` has quantized: ``x_fp8`` (M, K) e4m3,
    ``x_scale`` (M, ceil(K/128)) float32. Returns (M, N)."""
    N, K = _check_weight(w_fp8, w_scale)
    code = _check_out(out_dtype, bias, N)
    if x_fp8.ndim != 2 or x_fp8.shape[1] != K or x_fp8.dtype not in (torch.float8_e4m3fn, torch.uint8):
        raise ValueError(f"x_fp8 must be float8_e4m3fn of shape (M, {K}), got {x_fp8.dtype} {tuple(x_fp8.shape)}")
    M = x_fp8.shape[0]
    want = (M, -(-K // FP8_BLOCK))
    if tuple(x_scale.shape) != want or x_scale.dtype != torch.float32:
        raise ValueError(f"x_scale must be float32 of shape {want}, got {x_scale.dtype} {tuple(x_scale.shape)}")
    dev = A.cuda_index(x_fp8, x_scale, w_fp8, w_scale, bias)
    with A.on_device(dev):
        out = torch.empty((M, N), dtype=out_dtype, device=x_fp8.device)
        x_fp8, x_scale, w_fp8, w_scale = (t.contiguous() for t in (x_fp8, x_scale, w_fp8, w_scale))
        if bias is not None:
            bias = bias.contiguous()
        A.check(A.load().aeoq_fp8_block_gemm(x_fp8.data_ptr(), x_scale.data_ptr(), M, w_fp8.data_ptr(),
                                             w_scale.data_ptr(), N, K, A.ptr(bias), out.data_ptr(), code, N,
                                             A.err_ptr(dev), A.raw_stream(dev)))
    return out
