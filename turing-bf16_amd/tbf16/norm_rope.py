"""RMS norm of every query and key head and rotation by position, in one pass over both: what stands
between a model's projections and its attention. No counterpart in the reference.

    angles = torch.arange(n, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    cos, sin = angles.cos().float().cuda(), angles.sin().float().cuda()      # (n, R / 2), once
    q, k = tbf16.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions)

tbf16.autograd.qk_norm_rope is the same with gradients.
"""
from __future__ import annotations

import ctypes
import math

import torch

from ._ext import launch, lib, ptr

MAX_HEAD_DIM = 256


def _device(x, *others) -> int:
    """The device of x (its index), which the others have to be on too."""
    dev = x.get_device()
    if dev < 0:
        raise ValueError("tbf16: expected tensors on a ROCm (cuda) device")
    for t in others:
        if t.get_device() != dev:
            raise ValueError(f"tbf16.qk_norm_rope: tensors on {t.device} and {x.device}")
    return dev


def _heads(x):
    """(x, its (b, s, h) strides) with heads the kernels read in place: x itself or a copy."""
    st = x.stride()
    if st[-1] != 1 or any(v & 7 for v in st[:-1]) or x.data_ptr() & 15:
        x = x.clone(memory_format=torch.contiguous_format)
        st = x.stride()
    return x, (ctypes.c_int64 * 3)(*((0, *st[:2]) if len(st) == 3 else st[:3]))


def _table(t):
    return t if t.is_contiguous() and not t.data_ptr() & 15 else t.clone(memory_format=torch.contiguous_format)


class Call:
    """The checked arguments of one call: what forward and backward have in common."""

    def __init__(self, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
        shape, kshape = q.shape, k.shape
        if len(shape) not in (3, 4) or shape[:-2] != kshape[:-2] or shape[-1] != kshape[-1] or not shape[-2] or not kshape[-2]:
            raise ValueError(f"tbf16.qk_norm_rope: q {tuple(shape)} and k {tuple(kshape)} are not ((B,) S, H, D) and "
                             "((B,) S, Hkv, D)")
        D = shape[-1]
        if D % 16 or not 0 < D <= MAX_HEAD_DIM:
            raise ValueError(f"tbf16.qk_norm_rope: head dim {D} is not a multiple of 16 up to {MAX_HEAD_DIM}")
        if q.dtype is not torch.bfloat16 or k.dtype is not torch.bfloat16:
            raise TypeError("tbf16.qk_norm_rope: expected bf16 q and k")
        if q_weight.shape != (D,) or k_weight.shape != (D,):
            raise ValueError(f"tbf16.qk_norm_rope: weights {tuple(q_weight.shape)} and {tuple(k_weight.shape)} are not ({D},)")
        if q_weight.dtype is not k_weight.dtype or q_weight.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError("tbf16.qk_norm_rope: expected weights both bf16 or both fp32")
        if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[0] == 0:
            raise ValueError(f"tbf16.qk_norm_rope: cos {tuple(cos.shape)} and sin {tuple(sin.shape)} are not tables of one "
                             "shape (positions, rotated dims / 2)")
        if cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
            raise TypeError("tbf16.qk_norm_rope: expected fp32 cos and sin")
        R = 2 * cos.shape[1]
        if R % 16 or not 0 < R <= D:
            raise ValueError(f"tbf16.qk_norm_rope: {R} rotated dims are not a multiple of 16 up to the head dim {D}")
        lead = shape[:-2]
        if positions.dtype is not torch.int32:
            raise TypeError("tbf16.qk_norm_rope: expected int32 positions")
        if positions.shape != lead and positions.shape != lead[1:]:
            raise ValueError(f"tbf16.qk_norm_rope: positions {tuple(positions.shape)} for tokens {tuple(lead)}")
        if not 0.0 <= eps < math.inf:
            raise ValueError(f"tbf16.qk_norm_rope: eps {eps}")
        _device(q, k, q_weight, k_weight, cos, sin, positions)
        self.B, self.S = (1, shape[0]) if len(lead) == 1 else lead
        self.tokens = self.B * self.S
        if self.tokens >= 2 ** 31:
            raise ValueError(f"tbf16.qk_norm_rope: {self.tokens} tokens")
        p_st = positions.stride()
        self.p_st = p_st if len(p_st) == 2 else (0, *p_st) if len(p_st) else (0, 0)
        (self.q, self.q_st), (self.k, self.k_st) = _heads(q), _heads(k)
        self.wq, self.wk, self.cos, self.sin = q_weight.contiguous(), k_weight.contiguous(), _table(cos), _table(sin)
        self.pos, self.eps, self.near, self.D, self.R = positions, float(eps), int(bool(interleaved)), D, R

    def sizes(self):
        return self.B, self.S, self.q.shape[-2], self.k.shape[-2], self.D

    def tail(self):
        return (self.wq.data_ptr(), self.wk.data_ptr(), int(self.wq.dtype is torch.float32), self.cos.data_ptr(),
                self.sin.data_ptr(), self.cos.shape[0], self.R, self.pos.data_ptr(), *self.p_st, self.eps, self.near)

    def forward(self):
        q, k = self.q, self.k
        yq, yk = q.new_empty(q.shape), k.new_empty(k.shape)
        if self.tokens:
            launch("tbf16_qk_norm_rope", q, q.data_ptr(), k.data_ptr(), *self.sizes(), self.q_st, self.k_st, *self.tail(),
                   yq.data_ptr(), yk.data_ptr())
        return yq, yk

    def backward(self, dyq, dyk, want_q, want_k, want_wq, want_wk):
        q, k = self.q, self.k
        _device(q, dyq, dyk)
        (dyq, dyq_st), (dyk, dyk_st) = _heads(dyq.to(torch.bfloat16)), _heads(dyk.to(torch.bfloat16))
        dq = q.new_empty(q.shape) if want_q else None
        dk = k.new_empty(k.shape) if want_k else None
        dwq = torch.empty_like(self.wq) if want_wq else None
        dwk = torch.empty_like(self.wk) if want_wk else None
        ws = None
        if want_wq or want_wk:
            with torch.cuda.device(q.device):
                wsb = lib().tbf16_qk_norm_rope_bwd_ws_bytes(self.B, self.S, self.D)
            ws = q.new_empty(wsb, dtype=torch.uint8)
        launch("tbf16_qk_norm_rope_bwd", q, q.data_ptr(), k.data_ptr(), dyq.data_ptr(), dyk.data_ptr(), *self.sizes(),
               self.q_st, self.k_st, dyq_st, dyk_st, *self.tail(), ptr(dq), ptr(dk), ptr(dwq), ptr(dwk), ptr(ws),
               0 if ws is None else ws.numel())
        return dq, dk, dwq, dwk


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps=1e-6, interleaved=False):
    """(q', k'): with u = x / sqrt(mean(x^2) + eps) over a head and z = u * weight, the first R
    elements of z rotated by the token's position p in pairs (i, i + R / 2), or neighbours (2 i, 2 i + 1) where
    `interleaved`: (z_i cos[p, i] - z_j sin[p, i], z_j cos[p, i] + z_i sin[p, i]); elements from R on as they are.

    q bf16 (S, H, D) or (B, S, H, D), k the same with Hkv heads, any strides (views of one projection's
    output); weights (D,) bf16 or fp32; cos, sin fp32 (positions, R / 2); positions int32 (S,), or (B, S).
    D and R multiples of 16, D up to 256, R up to D. Returns contiguous bf16 tensors, rounded once from
    fp32. Tokens of a negative position are padding and give zeros; a position past the tables has no
    angle and gives NaN, as does a head of zeros without an eps. Inference only; gradients:
    tbf16.autograd.qk_norm_rope."""
    return Call(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved).forward()
