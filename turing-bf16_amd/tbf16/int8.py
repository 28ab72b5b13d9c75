"""Linears in 8-bit integers with one scale per token and per output channel.

x is quantised per row inside the call, W once by prepare_weight_i8; the products are summed
exactly in int32 on the i8 MFMA, and the epilogue applies both scales and the bias in fp32
with one rounding to bf16:

    sx[m] = max_k |x[m, k]| / 127        qx = rint(127 x / max_k |x|)   (ties to even)
    y[m, n] = (sum_k qx[m, k] w8[n, k]) * sx[m] * ws[n] + bias[n]

Beside scaled_linear, which keeps every bit of bf16: half its weight bytes (decoding) and
twice its matrix rate (prefill), for the rounding of x and W to 8 bits relative to each row's
maximum. The scales are fp32: rows of x with a maximum below 2^-95 lose bits of theirs, weight
rows above 2^110 overflow. No counterpart in the reference.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from ._ext import launch, lib, ptr
from .ops import _bias_bf16

# int32 sums of K products of two codes of magnitude at most 127 (TBF16_I8_MAX_K)
MAX_K = 131072


def _up(n, mult):
    return n + (-n) % mult


def _device(x, *others) -> int:
    """The device of x (its index), which the others have to be on too."""
    dev = x.get_device()
    if dev < 0:
        raise ValueError("tbf16: expected tensors on a ROCm (cuda) device")
    for t in others:
        if t.get_device() != dev:
            raise ValueError(f"tbf16.int8_linear: tensors on {t.device} and {x.device}")
    return dev


def _rows(x, K):
    """(x, its row stride) with columns side by side and rows apart (a single row's stride does
    not matter): x itself or a copy."""
    ld, step = x.stride()
    if (step == 1 or K == 1) and ld >= K:
        return x, ld
    if (step == 1 or K == 1) and x.shape[0] == 1:
        return x, K
    x = x.contiguous()
    return x, max(x.stride(0), K)


def quantize_rows_i8(x: torch.Tensor):
    """bf16 (R, K) -> (int8 (R, K), fp32 (R,) scales): codes rint(127 x / a) and a / 127, a the
    row's max |x|. The exact quotient decides, ties go to even. A row of zeros has scale 0; a
    row with an infinity or a NaN, which 8 bits cannot hold, zero codes and a NaN scale. The
    codes are a view of rows padded with zeros to a multiple of 16."""
    if x.dim() != 2:
        raise ValueError(f"tbf16.quantize_rows_i8: expected (R, K), got {tuple(x.shape)}")
    if x.dtype != torch.bfloat16:
        raise TypeError("tbf16.quantize_rows_i8: expected bf16")
    _device(x)
    R, K = x.shape
    if K > MAX_K:
        raise ValueError(f"tbf16.quantize_rows_i8: K = {K} is above {MAX_K}, int32 sums could overflow")
    x, ld = _rows(x, K)
    y = torch.empty((R, _up(K, 16)), device=x.device, dtype=torch.int8)
    scale = torch.empty((R,), device=x.device, dtype=torch.float32)
    if R:
        launch("tbf16_quantize_rows_i8", x, ptr(x), R, K, ld, ptr(y), y.stride(0), ptr(scale))
    return (y if y.shape[1] == K else y[:, :K]), scale


def prepare_weight_i8(w: torch.Tensor):
    """nn.Linear weight (N, K) bf16 -> (int8 (N, K), fp32 (N,) scales), once per weight:
    quantize_rows_i8 of its rows."""
    return quantize_rows_i8(w)


def _weight_rows(w8, K):
    """(w8, its row stride) with rows the kernels read in place: 16-byte aligned, apart by a
    multiple of 16 and readable up to K rounded up to 128 or to the next row (what
    prepare_weight_i8 returns); else a padded copy."""
    ld, step = w8.stride()
    if (step == 1 or K == 1) and not ld & 15 and K <= ld < 1 << 23 and not w8.data_ptr() & 15:
        if ld == K or (w8.untyped_storage().nbytes()
                       >= w8.storage_offset() + (w8.shape[0] - 1) * ld + min(ld, _up(K, 128))):
            return w8, ld
    w8 = F.pad(w8, (0, -K % 16)) if K % 16 else w8.clone(memory_format=torch.contiguous_format)
    return w8, _up(K, 16)


def padded_rows(w8: torch.Tensor) -> torch.Tensor:
    """An int8 weight (N, K) whose rows int8_linear reads in place: w8 itself, or a copy with padded
    rows (a weight that was moved, or loaded from elsewhere, has lost what prepare_weight_i8 gave it)."""
    K = w8.shape[1]
    rows = w8 if K == 0 else _weight_rows(w8, K)[0]
    return w8 if rows is w8 else rows[:, :K]


# tbf16_linear_i8's workspace bytes per (device, M, K, N): its choice of kernel counts the
# device's CUs, so it is asked on the tensors' device, once
_WS_BYTES: dict = {}


def _ws_bytes(dev: int, *sizes: int) -> int:
    key = (dev, sizes)
    n = _WS_BYTES.get(key)
    if n is None:
        if len(_WS_BYTES) > 4096:
            _WS_BYTES.clear()
        with torch.cuda.device(dev):
            n = _WS_BYTES[key] = int(lib().tbf16_linear_i8_ws_bytes(*sizes))
    return n


def int8_linear(x: torch.Tensor, w8: torch.Tensor, w_scale: torch.Tensor, bias=None):
    """y = x @ W^T + b for bf16 x (..., K), with W given by prepare_weight_i8 (its scales in fp32:
    rounded ones are refused). Returns bf16 (..., N). Rows of x with an infinity or a NaN give NaN. Inference only."""
    if x.dtype != torch.bfloat16:
        raise TypeError("tbf16.int8_linear: expected bf16 x")
    if w8.dtype != torch.int8 or w8.dim() != 2:
        raise TypeError("tbf16.int8_linear: expected an int8 weight (N, K)")
    shape = x.shape
    if len(shape) == 0:
        raise ValueError("tbf16.int8_linear: x has no dimension")
    K, (N, Kw) = shape[-1], w8.shape
    if Kw != K:
        raise ValueError(f"tbf16.int8_linear: x has K={K}, weight has K={Kw}")
    if K > MAX_K:
        raise ValueError(f"tbf16.int8_linear: K = {K} is above {MAX_K}, int32 sums could overflow")
    if w_scale.dtype != torch.float32 and w_scale.dtype != torch.float64:
        raise TypeError(f"tbf16.int8_linear: expected fp32 scales, got {w_scale.dtype}")
    if w_scale.numel() != N:
        raise ValueError(f"tbf16.int8_linear: {w_scale.numel()} scales for {N} channels")
    dev = _device(x, w8, w_scale)
    b = None if bias is None else _bias_bf16(bias, N, x.device)
    x2 = x if len(shape) == 2 else x.reshape(math.prod(shape[:-1]), K)
    M = x2.shape[0]
    if K == 0:
        y = torch.zeros((M, N), device=x.device, dtype=torch.bfloat16)
        return (y if b is None else y + b).reshape(*shape[:-1], N)
    Np = _up(N, 8)
    y = x.new_empty((M, Np))
    if M and N:
        x2, ldx = _rows(x2, K)
        w8, ldw = _weight_rows(w8, K)
        ws = w_scale if w_scale.dtype == torch.float32 and w_scale.is_contiguous() else w_scale.float().contiguous()
        wsb = _ws_bytes(dev, M, K, N)
        work = x.new_empty(wsb, dtype=torch.uint8) if wsb else None
        launch("tbf16_linear_i8", x2, x2.data_ptr(), M, K, ldx, w8.data_ptr(), N, ldw, ws.data_ptr(), ptr(b), y.data_ptr(),
               Np, ptr(work), wsb)
    if Np != N:
        y = y[:, :N]
    return y if len(shape) == 2 else y.reshape(*shape[:-1], N)
