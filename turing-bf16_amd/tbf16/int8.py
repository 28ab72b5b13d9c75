"""Linears in 8-bit integers with one scale per token and per output channel.

x is quantised per row inside the call, W once by prepare_weight_i8; the products are summed
exactly in int32 on the i8 MFMA, and the epilogue applies both scales and the bias in fp32
with one rounding to bf16:

    sx[m] = max_k |x[m, k]| / 127        qx = rint(127 x / max_k |x|)   (ties to even)
    y[m, n] = (sum_k qx[m, k] w8[n, k]) * sx[m] * ws[n] + bias[n]

Beside scaled_linear, which keeps every bit of bf16: half its weight bytes (decoding) and
twice its matrix rate (prefill), for the rounding of x and W to 8 bits relative to each row's
maximum. No counterpart in the reference.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from ._ext import launch, lib, ptr
from .ops import _bias_bf16, _dev_check

# int32 sums of K products of two codes of magnitude at most 127 (TBF16_I8_MAX_K)
MAX_K = 131072


def _up(n, mult):
    return n + (-n) % mult


def _rows(x):
    """x with its columns side by side and rows apart (a single row's stride does not matter)."""
    return x if (x.stride(1) == 1 or x.shape[1] == 1) and (x.stride(0) >= x.shape[1] or x.shape[0] == 1) else x.contiguous()


def quantize_rows_i8(x: torch.Tensor):
    """bf16 (R, K) -> (int8 (R, K), fp32 (R,) scales): codes rint(127 x / a) and a / 127, a the
    row's max |x|. The exact quotient decides, ties go to even. A row of zeros has scale 0; a
    row with an infinity or a NaN, which 8 bits cannot hold, zero codes and a NaN scale. The
    codes are a view of rows padded with zeros to a multiple of 16."""
    _dev_check(x)
    if x.dim() != 2:
        raise ValueError(f"tbf16.quantize_rows_i8: expected (R, K), got {tuple(x.shape)}")
    if x.dtype != torch.bfloat16:
        raise TypeError("tbf16.quantize_rows_i8: expected bf16")
    R, K = x.shape
    if K > MAX_K:
        raise ValueError(f"tbf16.quantize_rows_i8: K = {K} is above {MAX_K}, int32 sums could overflow")
    x = _rows(x)
    y = torch.empty((R, _up(K, 16)), device=x.device, dtype=torch.int8)
    scale = torch.empty((R,), device=x.device, dtype=torch.float32)
    if R:
        launch("tbf16_quantize_rows_i8", x, ptr(x), R, K, max(x.stride(0), K), ptr(y), y.stride(0), ptr(scale))
    return (y if y.shape[1] == K else y[:, :K]), scale


def prepare_weight_i8(w: torch.Tensor):
    """nn.Linear weight (N, K) bf16 -> (int8 (N, K), fp32 (N,) scales), once per weight:
    quantize_rows_i8 of its rows."""
    return quantize_rows_i8(w)


def _weight_rows(w8, K):
    """w8 with rows the kernels read in place: 16-byte aligned and padded to a multiple of
    16 inside their storage (what prepare_weight_i8 returns); else a padded copy."""
    N, Kp = w8.shape[0], _up(K, 16)
    ld = w8.stride(0)
    if (w8.stride(1) == 1 or K == 1) and ld % 16 == 0 and Kp <= ld < 1 << 23 and w8.data_ptr() % 16 == 0:
        if Kp == K or w8.untyped_storage().nbytes() >= w8.storage_offset() + (N - 1) * ld + Kp:
            return w8
    return F.pad(w8, (0, Kp - K)) if Kp != K else w8.clone(memory_format=torch.contiguous_format)


def int8_linear(x: torch.Tensor, w8: torch.Tensor, w_scale: torch.Tensor, bias=None):
    """y = x @ W^T + b for bf16 x (..., K), with W given by prepare_weight_i8. Returns bf16
    (..., N). Rows of x with an infinity or a NaN give NaN. Inference only."""
    _dev_check(x, w8, w_scale)
    if x.dtype != torch.bfloat16:
        raise TypeError("tbf16.int8_linear: expected bf16 x")
    if w8.dtype != torch.int8 or w8.dim() != 2:
        raise TypeError("tbf16.int8_linear: expected an int8 weight (N, K)")
    K, (N, Kw) = x.shape[-1], w8.shape
    if Kw != K:
        raise ValueError(f"tbf16.int8_linear: x has K={K}, weight has K={Kw}")
    if K > MAX_K:
        raise ValueError(f"tbf16.int8_linear: K = {K} is above {MAX_K}, int32 sums could overflow")
    if w_scale.numel() != N:
        raise ValueError(f"tbf16.int8_linear: {w_scale.numel()} scales for {N} channels")
    if w8.device != x.device or w_scale.device != x.device:
        raise ValueError(f"tbf16.int8_linear: x on {x.device}, weight on {w8.device}, scales on {w_scale.device}")
    shape = x.shape[:-1]
    b = _bias_bf16(bias, N, x.device)
    M = math.prod(shape)
    if K == 0:
        y = torch.zeros((M, N), device=x.device, dtype=torch.bfloat16)
        return (y if b is None else y + b).reshape(*shape, N)
    x2 = x.reshape(M, K)
    Np = _up(N, 8)
    y = torch.empty((M, Np), device=x.device, dtype=torch.bfloat16)
    if M and N:
        x2 = _rows(x2)
        w8, ws = _weight_rows(w8, K), w_scale.float().contiguous()
        wsb = lib().tbf16_linear_i8_ws_bytes(M, K, N)
        work = torch.empty((wsb,), device=x.device, dtype=torch.uint8)
        launch("tbf16_linear_i8", x2, ptr(x2), M, K, max(x2.stride(0), K), ptr(w8), N, w8.stride(0), ptr(ws), ptr(b), ptr(y),
               Np, ptr(work), wsb)
    return (y if Np == N else y[:, :N]).reshape(*shape, N)
